// w4_tc_kernel.cu -- the 4-bit projections for many rows of x, on tcgen05.
//
// x is 16-bit here, in rows that TMA can address: an fp32 x comes as its three
// bf16 parts, unaligned rows as copies (launch_rows).
// The same sums as w4_kernels.cu (integers q - z exact in the operand type,
// a group's products summed in fp32, the scale applied to the sum), with the
// roles of a tile spread over the warps of one CTA:
//   warps 0-3   unpack codes into the A operand: 128 weight rows x 128 inputs
//               in shared memory, 128-byte-swizzled K-major;
//   warp 4      brings the B operand: NB rows of x x 128 inputs, the same
//               layout, by TMA, which fills what lies outside x with zeros;
//   warp 7      issues the MMAs: each group of inputs into a fresh sum in
//               tensor memory, two or four of them in turn;
//   warps 8-15  read a finished group (lane = weight row) and add it, times
//               the row's scale, to fp32 sums in registers, while the next
//               group is multiplied.
// So the matrix instructions run back to back while the scaling, which they
// cannot do, follows a group behind.  A gated block's tile is 64 gate rows and
// the 64 up rows of the same outputs, which meet in shared memory at the end.
// Few tiles: a cluster of CTAs shares a tile's inputs and adds its sums by
// DSMEM in rank order.
//
// An M = 128, K = 16 MMA takes 48, 64 and 128 clocks for 64, 128 and 256 columns
// (back to back), and unpacking a span costs the same for each, so a tile has
// 256 columns where x has the rows for them; its sums then need 128 registers
// per scaling thread, which the unpacking and copying warps give up.
// Where the clocks of a CTA go (512 gated rows of 8960 x 1536, 12 spans; 256 rows
// of 1536 x 8960, 8 or 9 spans): a span 1820 / 1810, of which 1024 are the MMAs'; start and
// first span 4900 / 4700; joining the warps 2400 / 2400; the output pass 14100 / 10300.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "device_common.cuh"
#include "kvattn.h"
#include "kvattn_internal.h"
#include "projection.cuh"
#include "step_ops.h"
#include "tcgen05.cuh"
#include "w4_device.cuh"
#include "w4_internal.h"

namespace kvattn {

namespace {

constexpr int kStagesA = 2;   // written from registers, so little waits in them
template <int NB>
constexpr int kStagesB = NB == 256 ? 2 : 4;  // copies in flight
// Sums in tensor memory: groups that are committed and read together (a unit: the
// round trip between the MMAs and the reading is paid once for it), and units.
template <int NB, int GP>
constexpr int kUnit = GP < 256 / NB ? GP : 256 / NB;
template <int NB, int GP>
constexpr int kUnits = 512 / (kUnit<NB, GP> * NB) < 4 ? 512 / (kUnit<NB, GP> * NB) : 4;
constexpr int kAhead = 3;     // spans of codes in shared memory, per unpacking warp
constexpr int kCodes = 2 * 1024 + 128;  // a span of a warp's two tiles, and their zero points
constexpr int kThreads = 16 * 32;
constexpr int kMmaWarp = 7;
constexpr int kHalfA = 128 * 128;  // 64 inputs of 128 rows
// Registers of a thread of the unpacking, the copying and issuing and the two
// scaling warpgroups where a tile has 256 columns: what the launch has, dealt anew.
constexpr int kLaunchRegs = 65536 / kThreads, kRegs[3] = {104, 56, 176};
static_assert(kRegs[0] + kRegs[1] + 2 * kRegs[2] <= 4 * kLaunchRegs, "the scaling warps would wait for registers for good");

template <int NB>
struct Smem {
    static constexpr int kHalfB = NB * 128;
    static constexpr int kB = kStagesA * 2 * kHalfA;  // where the B stages start
    static constexpr int kRed = NB * 128 * 4;         // [column][row] sums, over the stages
    static constexpr int kRing = kB + kStagesB<NB> * 2 * kHalfB;  // the codes
    static_assert(kRed <= kRing, "");
    static constexpr int kBytes = 1024 + kRing + 4 * kAhead * kCodes;
};

struct Bars {
    uint64_t full_a[kStagesA], empty_a[kStagesA], full_b[4], empty_b[4], sum_full[4], sum_empty[4];
    uint64_t done;  // the MMAs in flight where a wait gave up
    uint32_t tmem;
    int failed;
};

// The public calls' status words, as a pool's: KV_ERR_TIMEOUT once a wait has run out, its CTA, where.
__device__ int g_step_status[3];

__device__ __noinline__ void gave_up(const W4Args& a, Bars* b) {
    int* const status = a.status ? a.status : g_step_status;
    if (atomicCAS(status, 0, KV_ERR_TIMEOUT) == 0) {
        status[1] = blockIdx.x;
        status[2] = 800;
    }
    *reinterpret_cast<volatile int*>(&b->failed) = 1;
}

// A whole warp's wait: all of its lanes, or none, go on.  The test without a
// suspend stands alone in front, as most waits end there: 512 gated rows 45.4 us,
// 48.5 with it behind the choice by the limit, 51.5 with the rest in a call.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Bars* b, const W4Args& a) {
    bool ok = mbar_test_wait(bar, parity) || (a.wait_limit > 0 && mbar_wait_bounded(bar, parity, a.wait_limit));
    if (!ok) gave_up(a, b);
    ok = ok && !*reinterpret_cast<volatile int*>(&b->failed);
    return __all_sync(0xffffffffu, ok);
}

// D (+)= A B.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// One lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one = 0;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n @p mov.u32 %0, 1;\n}" : "+r"(one));
    return one != 0;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// A box of 64 inputs x NB rows of x, zeros outside it.
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int k, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(k), "r"(row), "r"(smem_u32(bar))
        : "memory");
}

// BF: bf16 operands (else fp16).  GP: groups per span.  NB: columns (operand
// rows of x) of a tile.  GATED: two matrices.
template <int BF, int GP, int NB, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
    w4_tc_kernel(const __grid_constant__ W4Args a, const __grid_constant__ CUtensorMap xmap) {
    using SM = Smem<NB>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Bars bars;
    // from lane 0, so that the roles part by uniform branches
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int cs = a.cs, rank = (int)blockIdx.x % cs;
    const int tile0 = (int)blockIdx.x / cs * (GATED ? 4 : 8);  // first 16-row tile
    const int m0 = blockIdx.y * a.rows, mrows = min(a.rows, a.M - m0);
    const int s0 = (int)((long long)a.S * rank / cs), s1 = (int)((long long)a.S * (rank + 1) / cs);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < kStagesA; ++i) {
            mbar_init(&bars.full_a[i], 4);
            mbar_init(&bars.empty_a[i], 1);
        }
        for (int i = 0; i < kStagesB<NB>; ++i) {
            mbar_init(&bars.full_b[i], 1);
            mbar_init(&bars.empty_b[i], 1);
        }
        for (int i = 0; i < kUnits<NB, GP>; ++i) {
            mbar_init(&bars.sum_full[i], 1);
            mbar_init(&bars.sum_empty[i], 8);
        }
        mbar_init(&bars.done, 1);
        bars.failed = 0;
    }
    fence_mbar_init();
    if (warp == kMmaWarp) {
        tmem_alloc(&bars.tmem, kUnits<NB, GP> * kUnit<NB, GP> * NB);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // tile i (0..7) of the CTA's rows
    auto tile_of = [&](int i) { return min(tile0 + (GATED ? i & 3 : i), a.T - 1); };
    auto mat_of = [&](int i) { return GATED ? i >> 2 : 0; };
    auto flushes = [&](int sp) { return sp == a.S - 1 ? a.last_groups : GP; };

    if (warp < 4) {
        // ---------------------------------------------------- A: unpack codes
        if (NB == 256) regs_down<kRegs[0]>();
        // A short loop on purpose: sixteen warps of four roles share the
        // instruction caches, and unrolling this role starved the others.
        const int g = lane >> 2, c = lane & 3, odd = g & 1;
        const uint8_t* src[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = warp * 2 + i;
            src[i] = reinterpret_cast<const uint8_t*>(a.codes[mat_of(t)]) + ((size_t)tile_of(t) * a.S + s0) * 1024 + lane * 16;
        }
        // zero points: lane l brings four bytes of group l / 4 % GP of tile l / (4 GP)
        const int zt = warp * 2 + (lane / (4 * GP) & 1), zg = lane / 4 % GP;
        const bool zeros = a.zeros[0] != nullptr;
        const uint8_t* zsrc = zeros && lane < 8 * GP ? a.zeros[mat_of(zt)] + ((size_t)tile_of(zt) * a.Q + (size_t)s0 * GP + zg) * 16 + (lane & 3) * 4
                                                     : nullptr;
        uint8_t* const ring = smem + SM::kRing + warp * (kAhead * kCodes);
        const uint32_t ring_s = smem_u32(ring);
        int fslot = 0, fsp = s0;
        auto fetch = [&]() {
            if (fsp < s1) {
                const uint32_t to = ring_s + fslot * kCodes + lane * 16;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    cp16(to + i * 1024, src[i]);
                    cp16(to + i * 1024 + 512, src[i] + 512);
                    src[i] += 1024;
                }
                if (zsrc) {
                    if (fsp * GP + zg < a.Q) cp4(ring_s + fslot * kCodes + 2048 + lane * 4, zsrc);
                    zsrc += GP * 16;
                }
                ++fsp;
            }
            cp_commit();
            fslot = fslot + 1 == kAhead ? 0 : fslot + 1;
        };
#pragma unroll
        for (int d = 0; d < kAhead - 1; ++d) fetch();
        // odd rows take the words of a pair in the other order, so that eight
        // lanes' stores fall into eight different 16-byte columns
        const uint32_t row0 = (uint32_t)(warp * 32 + g) * 128;
        const uint32_t chunk0 = (uint32_t)((odd * 4 + c) ^ g) << 4;
        uint2 z = zero_consts<BF>(8u);
        int st = 0, ph = 1, slot = 0;
        for (int sp = s0; sp < s1; ++sp) {
            cp_wait<kAhead - 2>();
            __syncwarp();  // zero points came by other lanes; the slot refilled next was read by all of them
            fetch();
            if (sp - s0 >= kStagesA && !wait_warp(&bars.empty_a[st], ph, &bars, a)) break;
            const uint8_t* from = ring + slot * kCodes;
            uint8_t* to = smem + st * (2 * kHalfA) + row0 + chunk0;
#pragma unroll 1
            for (int th = 0; th < 4; ++th) {  // tile, rows g or g + 8
                const uint4 w = *reinterpret_cast<const uint4*>(from + th * 512 + lane * 16);
                const uint32_t v[4] = {odd ? w.y : w.x, odd ? w.x : w.y, odd ? w.w : w.z, odd ? w.z : w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // word j here is inputs 32 (j ^ odd) ..
                    if (zeros && j % (4 / GP) == 0) {
                        const int q = GP == 4 ? j ^ odd : j / (4 / GP);
                        z = zero_consts<BF>(from[2048 + ((th >> 1) * GP + q) * 16 + g * 2 + (th & 1)] & 15u);
                    }
                    uint32_t p[4];
                    unpack<BF>(v[j], z, p);
                    // the pair's second word is four 16-byte columns on (or back): bit 6 of the address
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(reinterpret_cast<size_t>(to) ^ ((j & 1) << 6)) + (j >> 1) * kHalfA) =
                        make_uint4(p[0], p[1], p[2], p[3]);
                }
                to += 8 * 128;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.full_a[st]);
            if (++st == kStagesA) st = 0, ph ^= 1;
            slot = slot + 1 == kAhead ? 0 : slot + 1;
        }
        cp_wait<0>();
    } else if (warp < 8) {
        if (NB == 256) regs_down<kRegs[1]>();  // by the whole warpgroup, before its warps' roles part
        if (warp == 4) {
            // --------------------------------------- B: rows of x (5 and 6 idle)
            int st = 0, ph = 1, sp = s0;
            for (; sp < s1; ++sp) {
                if (sp - s0 >= kStagesB<NB> && !wait_warp(&bars.empty_b[st], ph, &bars, a)) break;
                if (lane == 0) {
                    const uint32_t dst = smem_u32(smem) + SM::kB + st * (2 * SM::kHalfB);
                    mbar_arrive_expect_tx(&bars.full_b[st], 2 * SM::kHalfB);
                    tma_rows(dst, &xmap, sp * 128, m0 * a.pieces, &bars.full_b[st]);
                    tma_rows(dst + SM::kHalfB, &xmap, sp * 128 + 64, m0 * a.pieces, &bars.full_b[st]);
                }
                __syncwarp();
                if (++st == kStagesB<NB>) st = 0, ph ^= 1;
            }
            // no copy outlives the CTA, wherever another warp gave up
            for (int i = max(sp - s0 - kStagesB<NB>, 0); i < sp - s0; ++i)
                mbar_wait_bounded(&bars.full_b[i % kStagesB<NB>], (i / kStagesB<NB>) & 1, kW4WaitLimit);
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------- MMA issue
            // The whole warp runs the loop and one lane issues: the operands of an
            // MMA live in uniform registers, which only uniform control flow fills
            // directly.
            constexpr uint32_t idesc = idesc_f16(BF, 128, NB, 0);
            const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0), d0 = __shfl_sync(0xffffffffu, tmem, 0);
            constexpr int kG = kUnit<NB, GP>, kN = kUnits<NB, GP>;
            int f = 0, sta = 0, stb = 0, pha = 0, phb = 0;  // units so far; stages and their phases
            bool ok = true;
            for (int sp = s0; ok && sp < s1; ++sp) {
                ok = wait_warp(&bars.full_b[stb], phb, &bars, a) && wait_warp(&bars.full_a[sta], pha, &bars, a);
                if (!ok) break;
                tc_fence_after();
                const int ua = __shfl_sync(0xffffffffu, sta, 0), ub = __shfl_sync(0xffffffffu, stb, 0);
                const uint64_t da = sdesc(base + ua * (2 * kHalfA), 16, 1024), db = sdesc(base + SM::kB + ub * (2 * SM::kHalfB), 16, 1024);
                const int nf = flushes(sp);
#pragma unroll
                for (int q0 = 0; q0 < GP; q0 += kG) {
                    if (q0 >= nf) break;
                    const int unit = __shfl_sync(0xffffffffu, f % kN, 0);
                    if (f >= kN) {
                        ok = wait_warp(&bars.sum_empty[unit], (f / kN - 1) & 1, &bars, a);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    if (elect_one()) {
#pragma unroll
                        for (int q = q0; q < q0 + kG; ++q) {
                            if (q >= nf) break;
#pragma unroll
                            for (int i = 0; i < 8 / GP; ++i) {
                                const int kk = q * (8 / GP) + i;  // 16 inputs: 32 bytes on (the descriptors count 16)
                                mma_ss(d0 + (unit * kG + q - q0) * NB, da + ((kk >> 2) * kHalfA + (kk & 3) * 32) / 16,
                                       db + ((kk >> 2) * SM::kHalfB + (kk & 3) * 32) / 16, idesc, i != 0);
                            }
                        }
                        tc_commit(&bars.sum_full[unit]);
                        if (q0 + kG >= nf) {
                            tc_commit(&bars.empty_a[ua]);
                            tc_commit(&bars.empty_b[ub]);
                        }
                    }
                    __syncwarp();
                    ++f;
                }
                if (++sta == kStagesA) sta = 0, pha ^= 1;
                if (++stb == kStagesB<NB>) stb = 0, phb ^= 1;
            }
            __syncwarp();
        }
    } else {
        // -------------------------------------------------- scale and accumulate
        if (NB == 256) regs_up<kRegs[2]>();
        const int quarter = warp & 3, half = (warp - 8) >> 2;
        const int r = quarter * 32 + lane;  // weight row of the CTA
        const __half* sc = a.scales[mat_of(r >> 4)] + (size_t)tile_of(r >> 4) * a.Q * 16 + (r & 7) * 2 + ((r >> 3) & 1);
        float acc[NB / 2];
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) acc[i] = 0.f;
        float next[GP];  // the scales of a span, loaded a span ahead
        auto load_scales = [&](int sp) {
#pragma unroll
            for (int q = 0; q < GP; ++q) next[q] = sp < s1 && sp * GP + q < a.Q ? __half2float(sc[(size_t)(sp * GP + q) * 16]) : 0.f;
        };
        load_scales(s0);
        bool ok = true;
        int f = 0;
        for (int sp = s0; ok && sp < s1; ++sp) {
            float now[GP];
#pragma unroll
            for (int q = 0; q < GP; ++q) now[q] = next[q];
            load_scales(sp + 1);
            const int nf = flushes(sp);
            constexpr int kG = kUnit<NB, GP>, kN = kUnits<NB, GP>;
            constexpr int kD = NB == 64 ? 2 : 1;  // 32 columns read while 32 are added, where registers allow
#pragma unroll
            for (int q0 = 0; q0 < GP; q0 += kG) {
                if (q0 >= nf) break;
                const int unit = f % kN;
                ok = wait_warp(&bars.sum_full[unit], (f / kN) & 1, &bars, a);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(unit * kG * NB + half * (NB / 2));
                constexpr int kReads = kG * (NB / 64);  // of 32 columns
                const int reads = min(kG, nf - q0) * (NB / 64);
                float d[kD][32];
                if (kD == 2) tmem_ld32(at, d[0]);
#pragma unroll
                for (int i = 0; i < kReads; ++i) {
                    if (i >= reads) break;
                    const int q = q0 + i / (NB / 64), b = i % (NB / 64);
                    if (kD == 1) tmem_ld32(at + (i / (NB / 64)) * NB + b * 32, d[0]);
                    tc_wait_ld();
                    if (kD == 2 && i + 1 < reads) tmem_ld32(at + ((i + 1) / (NB / 64)) * NB + (i + 1) % (NB / 64) * 32, d[(i + 1) % kD]);
                    if (i == reads - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars.sum_empty[unit]);
                    }
#pragma unroll
                    for (int c = 0; c < 32; ++c) acc[b * 32 + c] = fmaf(now[q], d[i % kD][c], acc[b * 32 + c]);
                }
                ++f;
            }
        }
        // every MMA has read its operands: the stages become the sums
        float* red = reinterpret_cast<float*>(smem) + (size_t)half * (NB / 2) * 128 + r;
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the other half's last group too
        if (ok)
#pragma unroll
            for (int i = 0; i < NB / 2; ++i) red[i * 128] = acc[i];
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (NB == 256) {  // every warp goes on with the registers of the launch
        if (warp >= 8) regs_down<kLaunchRegs>();
        else regs_up<kLaunchRegs>();
    }
    const bool failed = *reinterpret_cast<volatile int*>(&bars.failed) != 0;
    if (warp == kMmaWarp) {
        if (failed && elect_one()) {  // MMAs in flight end before their memory goes
            tc_commit(&bars.done);
            mbar_wait_bounded(&bars.done, 0, kW4WaitLimit);
        }
        __syncwarp();
        tmem_dealloc(tmem, kUnits<NB, GP> * kUnit<NB, GP> * NB);
    }
    if (cs > 1) cluster_sync();
    // finished outputs: a thread keeps its output n and walks the rows of x
    constexpr int kN = GATED ? 64 : 128, kStep = kThreads / kN;
    const int i = tid % kN, n = tile0 * 16 + i;
    if (!failed && n < a.N) {
        const int first = tid / kN + rank * kStep, step = cs * kStep;
        const float* red = reinterpret_cast<const float*>(smem) + first * a.pieces * 128 + i;
        // the finished sum at `at`: over the cluster, in rank order
        auto sum_at = [&](const float* at) {
            if (cs == 1) return *at;
            float v[8], y = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < cs ? ld_cluster_f32(cluster_map(smem_u32(at), k)) : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) y += v[k];
            return y;
        };
        auto sum = [&](const float* at) {  // over the parts of a row, the smallest first
            return a.pieces == 1 ? sum_at(at) : sum_at(at + 256) + sum_at(at + 128) + sum_at(at);
        };
        if (a.mode == W4_LINEAR || a.mode == W4_GATED) {
            with_type(a.out_dtype, [&](auto one) {
                using T = decltype(one);
                T* out = static_cast<T*>(a.out) + (size_t)(m0 + first) * a.ldo + n;
                const T* res = static_cast<const T*>(a.residual);
                if (res) res += (size_t)(m0 + first) * a.ldr + n;
                const float bias = !GATED && a.bias ? __ldg(a.bias + n) : 0.f;
#pragma unroll 4
                for (int m = first; m < mrows; m += step) {
                    float y = sum(red);
                    if (GATED) {
                        y = gated(y, sum(red + 64));
                    } else {
                        if (a.bias) y += bias;
                        if (res) y += to_float(*res), res += (size_t)step * a.ldr;
                    }
                    *out = from_float<T>(y);
                    out += (size_t)step * a.ldo;
                    red += step * a.pieces * 128;
                }
            });
        } else {
            for (int m = first; m < mrows; m += step, red += step * 128)
                w4_epilogue(a, m0 + m, n, sum(red), sum(red + (GATED ? 64 : 0)));
        }
    }
    if (cs > 1) cluster_sync();  // nobody leaves while its sums are read
}

// x as TMA sees it: [M][K] 16-bit values in boxes of nb rows x 64 inputs, 128-byte swizzle.
cudaError_t x_map(const W4Args& a, bool bf, int nb, CUtensorMap* map) {
    static void* const encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return fn;
    }();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.M * a.pieces}, strides[1] = {(cuuint64_t)a.ldx * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)nb}, step[2] = {1, 1};
    const CUresult r = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(encode)(
        map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(a.x), dims, strides,
        box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int BF, int GP, int NB, bool GATED>
cudaError_t launch_inst(const W4Args& a, int gx, int gy, cudaStream_t st) {
    auto fn = w4_tc_kernel<BF, GP, NB, GATED>;
    static SmemGrant grant;
    cudaError_t e = grant.raise(reinterpret_cast<const void*>(fn), Smem<NB>::kBytes);
    if (e != cudaSuccess) return e;
    if (NB == 256) {
        // built with fewer registers, the scaling warps' share would never come free
        static const int regs = [&] {
            cudaFuncAttributes f = {};
            return cudaFuncGetAttributes(&f, fn) == cudaSuccess ? f.numRegs : 0;
        }();
        if (regs < kLaunchRegs) return cudaErrorInvalidConfiguration;
    }
    CUtensorMap map = {};
    if ((e = x_map(a, BF != 0, NB, &map)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(gx * a.cs), (unsigned)gy);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<NB>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cs > 1 ? 2 : 1;
    return counted(cudaLaunchKernelEx(&cfg, fn, a, map));
}

template <int BF, int GP, int NB>
cudaError_t launch_gated(const W4Args& a, bool gated, int gx, int gy, cudaStream_t st) {
    return gated ? launch_inst<BF, GP, NB, true>(a, gx, gy, st) : launch_inst<BF, GP, NB, false>(a, gx, gy, st);
}

template <int BF, int GP>
cudaError_t launch_nb(const W4Args& a, int nb, bool gated, int gx, int gy, cudaStream_t st) {
    return nb == 64    ? launch_gated<BF, GP, 64>(a, gated, gx, gy, st)
           : nb == 128 ? launch_gated<BF, GP, 128>(a, gated, gx, gy, st)
                       : launch_gated<BF, GP, 256>(a, gated, gx, gy, st);
}

template <int BF>
cudaError_t launch_group(const W4Args& a, int group, int nb, bool gated, int gx, int gy, cudaStream_t st) {
    if (group == 128) return launch_nb<BF, 1>(a, nb, gated, gx, gy, st);
    if (group == 64) return launch_nb<BF, 2>(a, nb, gated, gx, gy, st);
    return launch_nb<BF, 4>(a, nb, gated, gx, gy, st);
}

}  // namespace

// The limit of the waits in launches from now on.
static std::atomic<long long> g_wait_limit{kW4WaitLimit};

void set_wait_limit(long long clocks) { g_wait_limit.store(clocks < 0 ? kW4WaitLimit : clocks); }

cudaError_t launch_w4_tc(W4Args a, int group, bool bf, int nw, cudaStream_t st) {
    const W4TcPlan p = w4_tc_plan(a.M, a.T, a.S, a.pieces, nw);
    a.rows = p.rows;
    a.cs = p.cs;
    a.last_groups = a.Q - (a.S - 1) * (128 / group);
    a.wait_limit = g_wait_limit.load();
    return bf ? launch_group<1>(a, group, p.nb, nw == 2, p.gx, p.gy, st)
              : launch_group<0>(a, group, p.nb, nw == 2, p.gx, p.gy, st);
}

// Rows of x as TMA can address them, ldp elements apart, zeros from K on:
// row m as rows 3 m .. 3 m + 2 of its parts (T float), or as it is.
template <class T>
__global__ void __launch_bounds__(256)
    rows_kernel(const T* __restrict__ x, long long ldx, int M, int K, uint16_t* __restrict__ to, int ldp) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int per = ldp / 8;  // eight elements at a time
    const bool wide = (reinterpret_cast<size_t>(x) & 15) == 0 && ldx * sizeof(T) % 16 == 0;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < (long long)M * per; u += (long long)gridDim.x * 256) {
        const long long m = u / per;
        const int k = (int)(u % per) * 8;
        const T* row = x + m * ldx + k;
        T v[8];
        if (wide && k + 8 <= K) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(v)[j] = __ldg(reinterpret_cast<const uint4*>(row) + j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < K ? __ldg(row + j) : T(0);
        }
        constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
        uint16_t p[kParts][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (kParts == 3) split3(v[j], p[0][j], p[1][j], p[2][j]);
            else p[0][j] = v[j];
        }
#pragma unroll
        for (int q = 0; q < kParts; ++q)
            *reinterpret_cast<uint4*>(to + (m * kParts + q) * ldp + k) =
                make_uint4(p[q][0] | (uint32_t)p[q][1] << 16, p[q][2] | (uint32_t)p[q][3] << 16,
                           p[q][4] | (uint32_t)p[q][5] << 16, p[q][6] | (uint32_t)p[q][7] << 16);
    }
}

template <class T>
cudaError_t launch_rows_t(const void* x, long long ldx, int M, int K, void* to, cudaStream_t st) {
    const int ldp = (K + 7) / 8 * 8;
    const long long blocks = ((long long)M * (ldp / 8) + 255) / 256;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min(blocks, 8ll * kSms));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return counted(cudaLaunchKernelEx(&cfg, rows_kernel<T>, static_cast<const T*>(x), ldx, M, K, static_cast<uint16_t*>(to), ldp));
}

cudaError_t launch_rows(bool f32, const void* x, long long ldx, int M, int K, void* to, cudaStream_t st) {
    return f32 ? launch_rows_t<float>(x, ldx, M, K, to, st) : launch_rows_t<uint16_t>(x, ldx, M, K, to, st);
}

cudaError_t step_status(int* status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_step_status, sizeof(int));
    if (e != cudaSuccess) return e;
    const int zeros[3] = {};
    if (*status) e = cudaMemcpyToSymbol(g_step_status, zeros, sizeof zeros);
    return e;
}

}  // namespace kvattn
