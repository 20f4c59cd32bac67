// logits_kernels.cu -- penalties, biases, grammar masks and the greedy choice
// on rows of logits (logits_adjust of step_ops.h) in one pass.
//
// Bound: the logits' bytes, read once and written once.  A cluster of CTAs
// shares a row, each with a contiguous range of tokens, taken a chunk at
// a time.  What the history and the bias list say of a chunk's tokens is
// gathered in shared memory first -- one word per token: bit 31 met in the
// prompt, the lower bits how often it was generated; and the last bias entry of each
// token -- by reading the whole list and keeping what falls into the chunk,
// with atomics whose order does not matter (or, integer add, max).  Then the
// chunk's logits pass through registers once, 16 bytes at a time, several
// loads in flight.  The CTAs' best keys meet in the first CTA of the cluster.
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
constexpr int kMaxCluster = 8;
// Tokens whose notes are in shared memory at a time: two CTAs per SM.
template <class L>
constexpr int kChunk = sizeof(L) == 2 ? 19200 : 14336;
constexpr int kU = 2;          // 16-byte loads in flight per thread

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

// 16 bytes that pass through once (they may be written through `out` later).
__device__ __forceinline__ uint4 ld16_once(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// What is done to a row's tokens; L: the type of a bias entry's number.
template <class L>
struct RowRules {
    float rep, pres, freq;
    const uint32_t* met;  // notes of the chunk's tokens, NULL: no history
    const L* last;        // last bias entry + 1, NULL: no biases
    const float* bias;
    const uint32_t* mask;
};

__device__ __forceinline__ void note_last(uint32_t* at, uint32_t entry) { atomicMax(at, entry); }
__device__ __forceinline__ void note_last(uint16_t* at, uint32_t entry) {
    unsigned short old = *reinterpret_cast<volatile uint16_t*>(at);
    while (old < entry) {
        const unsigned short seen = atomicCAS(reinterpret_cast<unsigned short*>(at), old, (unsigned short)entry);
        if (seen == old) break;
        old = seen;
    }
}

// N logits of a row, tokens t .. t + N - 1, entry i of the chunk's notes on.
template <class T, int N, class L>
__device__ __forceinline__ void adjust(const RowRules<L>& q, const T* in, T* out, int t, int i, float& top, int& at) {
    uint32_t ok = 0xFFFFFFFFu;
    if (q.mask) {
        const uint32_t w0 = __ldg(q.mask + (t >> 5)), sh = t & 31;
        ok = w0 >> sh;
        if (N > 1 && sh + N > 32) ok |= __ldg(q.mask + (t >> 5) + 1) << (32 - sh);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float l = Elem<T>::get(in[j]);
        if (q.met) {
            const uint32_t w = q.met[i + j];
            if (w) {
                l = l > 0.f ? __fdiv_rn(l, q.rep) : __fmul_rn(l, q.rep);
                const uint32_t count = w & 0x7FFFFFFFu;
                if (count) l = __fsub_rn(__fsub_rn(l, __fmul_rn(q.freq, (float)count)), q.pres);
            }
        }
        if (q.last && q.last[i + j]) l = __fadd_rn(l, __ldg(q.bias + q.last[i + j] - 1));
        if (!((ok >> j) & 1u)) l = -INFINITY;
        out[j] = Elem<T>::put(l);
        // the lowest token wins: a thread's tokens rise
        if (l > top) {
            top = l;
            at = t + j;
        }
    }
}

template <class T, class L>
__global__ void __launch_bounds__(kThreads, 2)
    logits_kernel(const __grid_constant__ logits_call q, int chunk) {
    constexpr int kVec = 16 / sizeof(T);
    extern __shared__ __align__(16) uint32_t notes[];  // [chunk] history words, then [chunk] bias entries + 1
    __shared__ unsigned long long s_best[kThreads / 32], s_rank[kMaxCluster];
    const int row = blockIdx.y, rank = blockIdx.x, nrank = gridDim.x, tid = threadIdx.x;
    const int V = q.vocab;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // every CTA of the cluster has to run before its shared memory is written to
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int slice = ((V + nrank - 1) / nrank + 31) & ~31;
    const int t0 = min(rank * slice, V), t1 = min(t0 + slice, V);
    const T* in = static_cast<const T*>(q.logits) + (size_t)row * q.ld_logits;
    T* out = static_cast<T*>(q.out) + (size_t)row * q.ld_out;
    RowRules<L> rules;
    rules.mask = q.mask ? q.mask + (size_t)row * q.ld_mask : nullptr;
    rules.rep = q.repetition ? __ldg(q.repetition + row) : 1.f;
    rules.pres = q.presence ? __ldg(q.presence + row) : 0.f;
    rules.freq = q.frequency ? __ldg(q.frequency + row) : 0.f;
    const Cut h = q.hist ? cut(q.hist_off, row, q.hist_n) : Cut{0, 0};
    const Cut e = q.bias_ids ? cut(q.bias_off, row, q.bias_n) : Cut{0, 0};
    const long long gen = h.a + (q.gen_from ? max(__ldg(q.gen_from + row), 0) : 0);
    uint32_t* met = notes;
    L* last = reinterpret_cast<L*>(notes + (q.hist ? chunk : 0));
    rules.met = h.b > h.a ? met : nullptr;
    rules.bias = q.bias + e.a;
    rules.last = e.b > e.a ? last : nullptr;
    // tokens before the first 16-byte boundary of the row; vectors need both rows to agree on it
    const int shift = (int)((16 - (reinterpret_cast<size_t>(in) & 15)) & 15) / (int)sizeof(T);
    const bool vec = ((reinterpret_cast<size_t>(in) ^ reinterpret_cast<size_t>(out)) & 15) == 0;
    float top = -FLT_MAX;
    int at = -1;

    for (int c0 = t0; c0 < t1; c0 += chunk) {
        const int n = min(chunk, t1 - c0);
        if (rules.met || rules.last) {
            __syncthreads();
            if (rules.met)
                for (int i = tid * 4; i < n; i += kThreads * 4) *reinterpret_cast<uint4*>(met + i) = make_uint4(0u, 0u, 0u, 0u);
            if (rules.last)
                for (int i = tid * (16 / (int)sizeof(L)); i < n; i += kThreads * (16 / (int)sizeof(L)))
                    *reinterpret_cast<uint4*>(last + i) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            for (long long i0 = h.a + tid; i0 < h.b; i0 += kThreads * 8) {
                int id[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) id[u] = i0 + u * kThreads < h.b ? __ldg(q.hist + i0 + u * kThreads) : -1;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int t = id[u] - c0;
                    if (id[u] >= 0 && (unsigned)t < (unsigned)n) {
                        // a common word comes often: only the first of its prompt entries writes
                        if (i0 + u * kThreads >= gen) atomicAdd(met + t, 1u);
                        else if (!*reinterpret_cast<volatile uint32_t*>(met + t)) atomicOr(met + t, 0x80000000u);
                    }
                }
            }
            for (long long i = e.a + tid; i < e.b; i += kThreads) {
                const int id = __ldg(q.bias_ids + i), t = id - c0;
                if (id >= 0 && (unsigned)t < (unsigned)n) note_last(last + t, (uint32_t)(i - e.a + 1));
            }
            __syncthreads();
        }
        const int end = c0 + n;
        int v0 = end, v1 = end;  // vectors cover [v0, v1)
        if (vec) {
            v0 = min(end, c0 + (shift - c0 % kVec + kVec) % kVec);
            v1 = v0 + (end - v0) / kVec * kVec;
        }
        for (int t = c0 + tid; t < v0; t += kThreads) adjust<T, 1, L>(rules, in + t, out + t, t, t - c0, top, at);
        for (int t = v0 + tid * kVec; t < v1; t += kThreads * kVec * kU) {
            uint4 x[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (t + u * kThreads * kVec < v1) x[u] = ld16_once(in + t + u * kThreads * kVec);
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int tu = t + u * kThreads * kVec;
                if (tu >= v1) break;
                uint4 y;
                adjust<T, kVec, L>(rules, reinterpret_cast<const T*>(&x[u]), reinterpret_cast<T*>(&y), tu, tu - c0, top, at);
                *reinterpret_cast<uint4*>(out + tu) = y;
            }
        }
        for (int t = v1 + tid; t < end; t += kThreads) adjust<T, 1, L>(rules, in + t, out + t, t, t - c0, top, at);
    }
    unsigned long long best = at < 0 ? 0 : key_of(top, at);
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
        for (int r = 0; r < nrank; ++r) best = s_rank[r] > best ? s_rank[r] : best;
        q.pick[row] = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

template <class T, class L>
cudaError_t launch_tl(const logits_call& c, cudaStream_t st) {
    // eight CTAs to a row, fewer where a CTA would have less than 2048 tokens
    const int n = c.vocab >= 16384 ? 8 : c.vocab >= 8192 ? 4 : c.vocab >= 4096 ? 2 : 1;
    const int slice = ((c.vocab + n - 1) / n + 31) & ~31;
    const int chunk = slice < kChunk<L> ? slice : kChunk<L>;
    const int smem = (c.hist ? chunk * 4 : 0) + (c.bias_ids ? chunk * (int)sizeof(L) : 0);
    static SmemGrant grant;
    const cudaError_t e = grant.raise(reinterpret_cast<const void*>(logits_kernel<T, L>), kChunk<L> * (4 + (int)sizeof(L)));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n, (unsigned)c.rows);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    // may start while the previous kernel of the stream ends: it waits for that kernel before it reads anything
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return counted(cudaLaunchKernelEx(&cfg, logits_kernel<T, L>, c, chunk));
}

// Entries of a bias list are numbered in 16 bits where their total allows it.
template <class T>
cudaError_t launch_t(const logits_call& c, cudaStream_t st) {
    return c.bias_n <= 65535 ? launch_tl<T, uint16_t>(c, st) : launch_tl<T, uint32_t>(c, st);
}

}  // namespace

cudaError_t launch_logits(const logits_call& c, cudaStream_t st) {
    if (c.dtype == STEP_F32) return launch_t<float>(c, st);
    if (c.dtype == STEP_F16) return launch_t<__half>(c, st);
    return launch_t<__nv_bfloat16>(c, st);
}

}  // namespace kvattn
