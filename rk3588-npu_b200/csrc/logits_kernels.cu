// logits_kernels.cu -- penalties, biases, grammar masks and the greedy choice
// on rows of logits (logits_adjust of step_ops.h) in one pass.
//
// Bound: the logits' bytes, read once and written once.  A cluster of CTAs
// shares a row, its tokens dealt out in blocks of kBlock (common words, which
// stand together, fall to all of them), a chunk at a time.  What the history
// says of a chunk's tokens is gathered in shared memory first -- one word per
// token: bit 31 met in the prompt, the lower bits how often it was generated;
// and the last bias entry of each token -- by reading the whole list and
// keeping what is the CTA's own, with atomics whose order does not matter (or,
// integer add, max).  Then the chunk's logits pass through registers once, 16
// bytes at a time, the first of them loaded before the notes are taken; only
// words with notes in them take the long way.  The CTAs' best keys meet in
// the first one.  Sending each id to its owner instead of reading the list in
// every CTA (a DSMEM reduction per id) was slower: 73 us against 46 us for 61
// histories of up to 32768 ids.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <limits.h>
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
constexpr int kMaxCluster = 16;
constexpr int kBlockBits = 8;
constexpr int kBlock = 1 << kBlockBits;  // tokens of a row dealt to a CTA at a time
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

// What is done to a row's tokens.
struct RowRules {
    float rep, inv, pres, freq;
    bool fast;  // rep and its reciprocal are far from the ends of the range
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

template <class L>
struct FourOf;
template <>
struct FourOf<uint16_t> { using type = uint2; };
template <>
struct FourOf<uint32_t> { using type = uint4; };
__device__ __forceinline__ bool nonzero(uint2 v) { return (v.x | v.y) != 0; }
__device__ __forceinline__ bool nonzero(uint4 v) { return (v.x | v.y | v.z | v.w) != 0; }

// l / rep, correctly rounded.  Where both are far from the ends of the range:
// a quotient by the correctly rounded reciprocal, corrected by its exact
// residual (Markstein: the result is the correctly rounded quotient unless
// the divisor's significand is all ones), without a branch or a call.
__device__ __forceinline__ float div_rep(const RowRules& q, float l) {
    const float a = l * q.inv, r = fmaf(fmaf(-a, q.rep, l), q.inv, a);
    const uint32_t e = (__float_as_uint(l) >> 23) & 255u;
    return q.fast && e - 40u < 176u ? r : __fdiv_rn(l, q.rep);
}

// One logit with its token's history word.
__device__ __forceinline__ float penalise(const RowRules& q, float l, uint32_t met) {
    const uint32_t count = met & 0x7FFFFFFFu;
    const float p = l > 0.f ? div_rep(q, l) : __fmul_rn(l, q.rep);
    const float c = __fsub_rn(__fsub_rn(p, __fmul_rn(q.freq, (float)count)), q.pres);
    return met ? (count ? c : p) : l;
}

// A logit by itself: the ends of a row, and rows whose addresses differ.
// Its adjusted value.
template <class T>
__device__ __forceinline__ float one_logit(const RowRules& q, const T* in, T* out, int t, uint32_t met, uint32_t last) {
    float l = penalise(q, Elem<T>::get(in[t]), met);
    if (last) l = __fadd_rn(l, __ldg(q.bias + last - 1));
    if (q.mask && !((__ldg(q.mask + (t >> 5)) >> (t & 31)) & 1u)) l = -INFINITY;
    out[t] = Elem<T>::put(l);
    return l;
}

template <class T, class L>
__global__ void __launch_bounds__(kThreads, 2)
    logits_kernel(const __grid_constant__ logits_call q, int chunk, int lrank /* log2 CTAs per row */) {
    constexpr int kVec = 16 / sizeof(T);
    extern __shared__ __align__(16) uint32_t notes[];  // [chunk] history words, then [chunk] bias entries + 1
    __shared__ unsigned long long s_best[kThreads / 32], s_rank[kMaxCluster];
    const int row = blockIdx.y, rank = blockIdx.x, nrank = 1 << lrank, tid = threadIdx.x;
    const int V = q.vocab;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // every CTA of the cluster has to run before its shared memory is written to
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const T* in = static_cast<const T*>(q.logits) + (size_t)row * q.ld_logits;
    T* out = static_cast<T*>(q.out) + (size_t)row * q.ld_out;
    // Token t stands at position t + off, so that multiples of kVec are on
    // 16-byte boundaries; block b of positions belongs to CTA b % nrank, where
    // position p is number (b / nrank) kBlock + p % kBlock.
    const int off = (int)((reinterpret_cast<size_t>(in) & 15) / sizeof(T));
    const bool vec = ((reinterpret_cast<size_t>(in) ^ reinterpret_cast<size_t>(out)) & 15) == 0;
    const int blocks = (V + off + kBlock - 1) / kBlock;
    const int own = ((blocks + nrank - 1) >> lrank) * kBlock;  // positions per CTA (the same for all; the last ones may be past the row)
    constexpr int kStep = kThreads * kVec;  // positions of a CTA per access of all its threads: whole blocks
    static_assert(kStep % kBlock == 0, "a thread's tokens are kStep << lrank apart");
    const int first = ((tid * kVec / kBlock << lrank) + rank) * kBlock + tid * kVec % kBlock - off;  // token of number tid * kVec
    const int apart = kStep << lrank;  // tokens from one access of a thread to its next
    // accesses of this thread among positions [c0, c0 + n) that lie inside the row: [from, to) of `all`
    struct Part {
        int t0, from, to, all;
    };
    auto part_of = [&](int c0, int n) {
        Part p;
        p.t0 = first + (c0 << lrank);
        p.all = tid * kVec < n ? (n - tid * kVec + kStep - 1) / kStep : 0;
        p.from = p.t0 < 0 ? 1 : 0;
        p.to = vec && V - kVec >= p.t0 ? min(p.all, (V - kVec - p.t0) / apart + 1) : 0;
        p.from = min(p.from, p.to);
        return p;
    };
    // an access's logits and, where there is a mask, the word with its first bit
    uint4 x[kU];
    uint32_t bits[kU];
    const uint32_t* const mask = q.mask ? q.mask + (size_t)row * q.ld_mask : nullptr;
    auto load = [&](int t, int left) {
#pragma unroll
        for (int u = 0; u < kU; ++u)
            if (u < left) {
                x[u] = ld16_once(in + t + u * apart);
                if (mask) bits[u] = __ldg(mask + ((t + u * apart) >> 5));
            }
    };
    Part part = part_of(0, min(chunk, own));
    load(part.t0 + part.from * apart, part.to - part.from);

    RowRules rules;
    rules.mask = mask;
    rules.rep = q.repetition ? __ldg(q.repetition + row) : 1.f;
    rules.inv = __frcp_rn(rules.rep);
    const uint32_t rb = __float_as_uint(rules.rep);
    rules.fast = ((rb >> 23) & 255u) - 107u < 40u && (rb & 0x7FFFFFu) != 0x7FFFFFu;  // 2^-20 to 2^20
    rules.pres = q.presence ? __ldg(q.presence + row) : 0.f;
    rules.freq = q.frequency ? __ldg(q.frequency + row) : 0.f;
    const Cut h = q.hist ? cut(q.hist_off, row, q.hist_n) : Cut{0, 0};
    const Cut e = q.bias_ids ? cut(q.bias_off, row, q.bias_n) : Cut{0, 0};
    const int* hist = q.hist + h.a;
    const int hist_n = (int)min(h.b - h.a, (long long)INT_MAX), gen = q.gen_from ? max(__ldg(q.gen_from + row), 0) : 0;
    const int head = min((int)((16 - (reinterpret_cast<size_t>(hist) & 15)) & 15) / 4, hist_n);
    const int wide = (hist_n - head) / 4, tail = hist_n - head - 4 * wide;
    const uint32_t mine = (uint32_t)rank << kBlockBits, others = (uint32_t)(nrank - 1) << kBlockBits;
    const bool has_met = h.b > h.a, has_last = e.b > e.a;
    uint32_t* met = notes;
    L* last = reinterpret_cast<L*>(notes + (q.hist ? chunk : 0));
    rules.bias = q.bias + e.a;
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    float top = -FLT_MAX;
    int at = -1;

    for (int c0 = 0; c0 < own; c0 += chunk) {
        const int n = min(chunk, own - c0);
        if (has_met || has_last) {
            if (c0) __syncthreads();
            if (has_met)
                for (int i = tid * 4; i < n; i += kThreads * 4) *reinterpret_cast<uint4*>(met + i) = make_uint4(0u, 0u, 0u, 0u);
            if (has_last)
                for (int i = tid * (16 / (int)sizeof(L)); i < n; i += kThreads * (16 / (int)sizeof(L)))
                    *reinterpret_cast<uint4*>(last + i) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            // the history, 16 bytes at a time from its first boundary on
            auto note = [&](int id, int k) {  // entry k of the row's history
                const uint32_t p = (uint32_t)(id + off);
                if ((p ^ mine) & others) return;
                const uint32_t i = (p >> (kBlockBits + lrank) << kBlockBits | (p & (kBlock - 1))) - (uint32_t)c0;
                if ((uint32_t)id >= (uint32_t)V || i >= (uint32_t)n) return;
                // a common word comes often: only the first of its prompt entries writes
                if (k >= gen) atomicAdd(met + i, 1u);
                else if (!*reinterpret_cast<volatile uint32_t*>(met + i)) atomicOr(met + i, 0x80000000u);
            };
            if (tid < head) note(__ldg(hist + tid), tid);
            if (tid < tail) note(__ldg(hist + head + 4 * wide + tid), head + 4 * wide + tid);
            for (int v = tid; v < wide; v += kThreads * 2) {
                int4 id[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    id[u] = v + u * kThreads < wide ? __ldg(reinterpret_cast<const int4*>(hist + head) + v + u * kThreads) : make_int4(-1 - off, -1 - off, -1 - off, -1 - off);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int k = head + 4 * (v + u * kThreads);
                    note(id[u].x, k);
                    note(id[u].y, k + 1);
                    note(id[u].z, k + 2);
                    note(id[u].w, k + 3);
                }
            }
            for (long long i = e.a + tid; i < e.b; i += kThreads) {
                const int id = __ldg(q.bias_ids + i);
                if ((unsigned)id >= (unsigned)V) continue;
                const int p = id + off, b = p / kBlock, at_i = (b >> lrank) * kBlock + p % kBlock - c0;
                if ((b & (nrank - 1)) == rank && (unsigned)at_i < (unsigned)n) note_last(last + at_i, (uint32_t)(i - e.a + 1));
            }
            __syncthreads();
        }
        if (c0) part = part_of(c0, n);
        const int i_first = tid * kVec;
        auto alone = [&](int a) {  // access a, token by token
#pragma unroll 1
            for (int j = 0; j < kVec; ++j) {
                const int t = part.t0 + a * apart + j, i = i_first + a * kStep + j;
                if (t < 0 || t >= V) continue;
                const float l = one_logit<T>(rules, in, out, t, has_met ? met[i] : 0u, has_last ? (uint32_t)last[i] : 0u);
                if (l > top || (l == top && t < at)) {
                    top = l;
                    at = t;
                }
            }
        };
        T* pout = out + part.t0 + part.from * apart;
        int t = part.t0 + part.from * apart, i = i_first + part.from * kStep;
        const uint32_t sh = t & 31;  // the same for all of a thread's accesses
#pragma unroll 1
        for (int left = part.to - part.from; left > 0; left -= kU) {
            if (c0 || left != part.to - part.from) load(t, left);
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (u >= left) break;
                float l[kVec];
                const T* from = reinterpret_cast<const T*>(&x[u]);
#pragma unroll
                for (int j = 0; j < kVec; ++j) l[j] = Elem<T>::get(from[j]);
                if (has_met) {
#pragma unroll
                    for (int j = 0; j < kVec; j += 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(met + i + j);
                        if (v.x | v.y | v.z | v.w) {
                            l[j] = penalise(rules, l[j], v.x);
                            l[j + 1] = penalise(rules, l[j + 1], v.y);
                            l[j + 2] = penalise(rules, l[j + 2], v.z);
                            l[j + 3] = penalise(rules, l[j + 3], v.w);
                        }
                    }
                }
                if (has_last) {
#pragma unroll
                    for (int j = 0; j < kVec; j += 4)
                        if (nonzero(*reinterpret_cast<const typename FourOf<L>::type*>(last + i + j))) {
#pragma unroll
                            for (int k = j; k < j + 4; ++k)
                                if (last[i + k]) l[k] = __fadd_rn(l[k], __ldg(rules.bias + last[i + k] - 1));
                        }
                }
                if (mask) {
                    uint32_t ok = bits[u] >> sh;
                    if (sh + kVec > 32) ok |= __ldg(mask + (t >> 5) + 1) << (32 - sh);
#pragma unroll
                    for (int j = 0; j < kVec; ++j) l[j] = (ok >> j) & 1u ? l[j] : -INFINITY;
                }
                float most = l[0];
#pragma unroll
                for (int j = 1; j < kVec; ++j) most = fmaxf(most, l[j]);  // a NaN never counts
                if (most > top) {
                    // the lowest token wins: a thread's tokens rise
                    top = most;
#pragma unroll
                    for (int j = kVec - 1; j >= 0; --j) at = l[j] == most ? t + j : at;
                }
                union {
                    uint4 v;
                    T el[kVec];
                } y;
#pragma unroll
                for (int j = 0; j < kVec; ++j) y.el[j] = Elem<T>::put(l[j]);
                *reinterpret_cast<uint4*>(pout) = y.v;
                pout += apart;
                t += apart;
                i += kStep;
            }
        }
        // the ends of the row last: among equal values the lower token wins
#pragma unroll 1
        for (int a = 0; a < part.all; ++a) {
            if (a == part.from) a = part.to;
            if (a < part.all) alone(a);
        }
    }
    unsigned long long best = at < 0 ? 0 : key_of(top, at);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
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
    // CTAs per row: 8 blocks or more each, at most 16, and 8 where the rows fill the SMs
    const int blocks = (c.vocab + kBlock - 1) / kBlock + 1;
    int lrank = 0;
    while (lrank < (c.rows <= 16 ? 4 : 3) && (8 << lrank) < blocks) ++lrank;
    const int n = 1 << lrank;
    const int own = ((blocks + n - 1) >> lrank) * kBlock;  // at least what a CTA owns
    const int chunk = own < kChunk<L> ? own : kChunk<L>;
    const int smem = (c.hist ? chunk * 4 : 0) + (c.bias_ids ? chunk * (int)sizeof(L) : 0);
    static SmemGrant grant;
    const cudaError_t e = grant.raise(reinterpret_cast<const void*>(logits_kernel<T, L>), kChunk<L> * (4 + (int)sizeof(L)), true);
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
    return counted(cudaLaunchKernelEx(&cfg, logits_kernel<T, L>, c, chunk, lrank));
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
