// logits_kernels.cu -- penalties, biases, grammar masks and the greedy choice
// on rows of logits (logits_adjust of step_ops.h) in one pass.
//
// Bound: the logits' bytes, read once and written once.  A cluster of CTAs
// shares a row; each CTA owns a contiguous range of tokens, taken kChunk at a
// time.  What the history and the bias list say of a chunk's tokens is
// gathered in shared memory first -- one word per token: bit 31 met before,
// the lower bits how often it was generated; and the last bias entry of each
// token -- by reading the whole list and keeping what falls into the chunk,
// with atomics whose order does not matter (or, integer add, max).  Then the
// chunk's logits pass through registers once.  The CTAs' best keys meet in
// the first CTA of the cluster.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "device_common.cuh"
#include "kvattn.h"
#include "kvattn_internal.h"
#include "step_ops.h"
#include "w4_internal.h"

namespace kvattn {

namespace {

constexpr int kThreads = 512;
constexpr int kCluster = 8;
constexpr int kChunk = 8192;  // tokens whose notes are in shared memory at a time

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// Largest value above -FLT_MAX at its lowest token: order-preserving bits of
// the value, then the complement of the token; 0 for none.  -0 counts as +0.
__device__ __forceinline__ unsigned long long key_of(float f, int t) {
    if (!(f > -FLT_MAX)) return 0;
    const uint32_t u = __float_as_uint(__fadd_rn(f, 0.f));
    const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)ord << 32) | (0xFFFFFFFFu - (uint32_t)t);
}

struct Cut {
    long long a, b;
};
// The range of row r in a list of n entries cut by off.
__device__ __forceinline__ Cut cut(const int* off, int r, long long n) {
    const long long a = min(max((long long)__ldg(off + r), 0ll), n), b = min(max((long long)__ldg(off + r + 1), a), n);
    return {a, b};
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    logits_kernel(const __grid_constant__ logits_call q) {
    extern __shared__ __align__(16) uint32_t notes[];  // [kChunk] history, then [kChunk] bias entries + 1
    __shared__ unsigned long long s_best[kThreads / 32], s_rank[kCluster];
    const int row = blockIdx.y, rank = cluster_rank(), tid = threadIdx.x;
    const int V = q.vocab;
    const int slice = ((V + kCluster - 1) / kCluster + 31) & ~31;
    const int t0 = min(rank * slice, V), t1 = min(t0 + slice, V);
    const T* in = static_cast<const T*>(q.logits) + (size_t)row * q.ld_logits;
    T* out = static_cast<T*>(q.out) + (size_t)row * q.ld_out;
    const uint32_t* mask = q.mask ? q.mask + (size_t)row * q.ld_mask : nullptr;
    const float rep = q.repetition ? __ldg(q.repetition + row) : 1.f;
    const float pres = q.presence ? __ldg(q.presence + row) : 0.f;
    const float freq = q.frequency ? __ldg(q.frequency + row) : 0.f;
    const Cut h = q.hist ? cut(q.hist_off, row, q.hist_n) : Cut{0, 0};
    const Cut e = q.bias_ids ? cut(q.bias_off, row, q.bias_n) : Cut{0, 0};
    const long long gen = h.a + (q.gen_from ? max(__ldg(q.gen_from + row), 0) : 0);
    uint32_t* met = notes;
    uint32_t* last = notes + (q.hist ? kChunk : 0);
    unsigned long long best = 0;
    // every CTA of the cluster has to run before its shared memory is written to
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");

    for (int c0 = t0; c0 < t1; c0 += kChunk) {
        const int n = min(kChunk, t1 - c0);
        if (h.b > h.a || e.b > e.a) {
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                if (h.b > h.a) met[i] = 0;
                if (e.b > e.a) last[i] = 0;
            }
            __syncthreads();
            for (long long i = h.a + tid; i < h.b; i += kThreads) {
                const int t = __ldg(q.hist + i) - c0;
                if ((unsigned)t < (unsigned)n) {
                    atomicOr(met + t, 0x80000000u);
                    if (i >= gen) atomicAdd(met + t, 1u);
                }
            }
            for (long long i = e.a + tid; i < e.b; i += kThreads) {
                const int t = __ldg(q.bias_ids + i) - c0;
                if ((unsigned)t < (unsigned)n) atomicMax(last + t, (uint32_t)(i - e.a + 1));
            }
            __syncthreads();
        }
        for (int i = tid; i < n; i += kThreads) {
            const int t = c0 + i;
            float l = Elem<T>::get(in[t]);
            if (h.b > h.a) {
                const uint32_t w = met[i];
                if (w) {
                    l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
                    const uint32_t count = w & 0x7FFFFFFFu;
                    if (count) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)count)), pres);
                }
            }
            if (e.b > e.a && last[i]) l = __fadd_rn(l, __ldg(q.bias + e.a + last[i] - 1));
            if (mask && !((__ldg(mask + (t >> 5)) >> (t & 31)) & 1u)) l = -INFINITY;
            out[t] = Elem<T>::put(l);
            const unsigned long long k = key_of(l, t);
            best = k > best ? k : best;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
        const uint32_t to = cluster_map(smem_u32(s_rank + rank), 0);
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to), "l"(best) : "memory");
    }
    cluster_sync();
    if (rank == 0 && tid == 0 && q.pick) {
        for (int r = 0; r < kCluster; ++r) best = s_rank[r] > best ? s_rank[r] : best;
        q.pick[row] = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

template <class T>
cudaError_t launch_t(const logits_call& c, cudaStream_t st) {
    const int smem = (c.hist ? kChunk * 4 : 0) + (c.bias_ids ? kChunk * 4 : 0);
    static SmemGrant grant;
    const cudaError_t e = grant.raise(reinterpret_cast<const void*>(logits_kernel<T>), 2 * kChunk * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCluster, (unsigned)c.rows);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return counted(cudaLaunchKernelEx(&cfg, logits_kernel<T>, c));
}

}  // namespace

cudaError_t launch_logits(const logits_call& c, cudaStream_t st) {
    if (c.dtype == STEP_F32) return launch_t<float>(c, st);
    if (c.dtype == STEP_F16) return launch_t<__half>(c, st);
    return launch_t<__nv_bfloat16>(c, st);
}

}  // namespace kvattn
