// step_ops.cu -- the C ABI of step_ops.h: argument checks and launches.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

#include "kvattn.h"
#include "kvattn_internal.h"
#include "step_ops.h"
#include "w4_internal.h"

using namespace kvattn;

namespace {

int sfail(int status, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return set_error(status, buf);
}

#define ST_OK(call)                \
    do {                           \
        int s_ = (call);           \
        if (s_ != KV_OK) return s_; \
    } while (0)

constexpr int kMaxDim = 1 << 30;   // outputs, inputs, tokens of one call
constexpr int kMaxRows = 1 << 19;  // rows of x of one call: 65535 passes of 10 hold them

bool aligned(const void* p, size_t n) { return (reinterpret_cast<size_t>(p) & (n - 1)) == 0; }
size_t esize(int dtype) { return dtype == STEP_F32 ? 4 : 2; }

int check_shape(int n, int k, int group) {
    if (n <= 0 || k <= 0 || n > kMaxDim || k > kMaxDim) return sfail(KV_ERR_INVAL, "a 4-bit matrix of %d x %d", n, k);
    if (group != 32 && group != 64 && group != 128)
        return sfail(KV_ERR_INVAL, "groups of %d inputs: 32, 64 or 128 are supported", group);
    return KV_OK;
}

int check_matrix(const w4_matrix* m, const char* what) {
    if (!m) return sfail(KV_ERR_INVAL, "NULL %s", what);
    ST_OK(check_shape(m->n, m->k, m->group));
    if (m->device < 0) return sfail(KV_ERR_INVAL, "%s: no device", what);
    if (!m->codes || !m->scales) return sfail(KV_ERR_INVAL, "%s: NULL codes or scales", what);
    if (!aligned(m->codes, 16) || !aligned(m->scales, 16) || !aligned(m->zeros, 16))
        return sfail(KV_ERR_INVAL, "%s: codes, scales and zero points need 16-byte alignment", what);
    return KV_OK;
}

// `rows` rows of `n` elements, `ld` apart: the bytes that they span, and whether
// any of them are another's.  Rows of one pitch may lie between the other's
// (columns of one buffer); where the pitches differ, spans that meet count as shared.
struct Range {
    size_t a, b;
    long long rows, width, pitch;
    Range(const void* p, long long rows, long long n, long long ld, size_t es)
        : a(reinterpret_cast<size_t>(p)), b(a + (rows > 0 ? (size_t)((rows - 1) * ld + n) * es : 0)), rows(rows),
          width(n * (long long)es), pitch(ld * (long long)es) {}
    bool meets(const Range& o) const {
        if (a >= o.b || o.a >= b) return false;
        if (pitch != o.pitch || pitch <= 0) return true;
        // row i here and row j there meet where t = i - j has  t pitch < d + o.width  and  t pitch > d - width
        const long long d = (long long)(o.a - a);
        auto below = [&](long long v) { return v >= 0 ? v / pitch : -((-v + pitch - 1) / pitch); };  // floor(v / pitch)
        const long long first = std::max(below(d - width) + 1, 1 - o.rows), last = std::min(-below(-(d + o.width)) - 1, rows - 1);
        return first <= last;
    }
};

int check_dtype(int dtype, const char* what) {
    if (dtype != STEP_F16 && dtype != STEP_BF16 && dtype != STEP_F32)
        return sfail(KV_ERR_INVAL, "%s: unsupported element type %d", what, dtype);
    return KV_OK;
}

int check_rows(const w4_matrix& w, const void* x, int x_dtype, int m, long long ldx, const void* out, int out_dtype,
               long long ldo) {
    ST_OK(check_dtype(x_dtype, "x"));
    ST_OK(check_dtype(out_dtype, "out"));
    if (m < 0) return sfail(KV_ERR_INVAL, "%d rows", m);
    if (ldx < w.k || ldo < w.n)
        return sfail(KV_ERR_INVAL, "rows %lld / %lld apart are shorter than %d inputs / %d outputs", ldx, ldo, w.k, w.n);
    if (ldx > (1ll << 40) || ldo > (1ll << 40)) return sfail(KV_ERR_INVAL, "rows too far apart");
    if (m == 0) return KV_OK;
    if (!x || !out) return sfail(KV_ERR_INVAL, "NULL x or out");
    if (!aligned(x, esize(x_dtype)) || !aligned(out, esize(out_dtype)))
        return sfail(KV_ERR_INVAL, "x or out is not aligned to its element");
    if (m > kMaxRows) return sfail(KV_ERR_RANGE, "%d rows in one call (at most %d)", m, kMaxRows);
    if (Range(x, m, w.k, ldx, esize(x_dtype)).meets(Range(out, m, w.n, ldo, esize(out_dtype))))
        return sfail(KV_ERR_INVAL, "out overlaps x");
    return KV_OK;
}

void set_x(W4Args& a, const void* x, int x_dtype, int m, long long ldx) {
    a.x = x;
    a.ldx = ldx;
    a.M = m;
    a.in = x_dtype == STEP_F32 ? W4_X_F32 : W4_X_16;
    a.pieces = x_dtype == STEP_F32 ? 3 : 1;
}

size_t work_bytes(int n, int k, int group, int x_dtype, int m, int gated) {
    const int pieces = x_dtype == STEP_F32 ? 3 : 1;
    return w4_use_tc(m, (n + 15) / 16, (k + 127) / 128, pieces, gated ? 2 : 1, group) ? w4_rows_bytes(m, k, pieces) : 0;
}

int check_work(const w4_matrix& w, const void* x, int x_dtype, int m, long long ldx, const void* out, int out_dtype,
               long long ldo, int gated, const void* work) {
    if (!work || m == 0) return KV_OK;
    if (!aligned(work, 16)) return sfail(KV_ERR_INVAL, "scratch needs 16-byte alignment");
    const Range r(work, 1, (long long)work_bytes(w.n, w.k, w.group, x_dtype, m, gated), 0, 1);
    if (r.meets(Range(x, m, w.k, ldx, esize(x_dtype))) || r.meets(Range(out, m, w.n, ldo, esize(out_dtype))))
        return sfail(KV_ERR_INVAL, "scratch overlaps x or out");
    return KV_OK;
}

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return KV_OK;
    return sfail(KV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(taken(e)));
}

}  // namespace

extern "C" {

int w4_sizes(int n, int k, int group, size_t* codes, size_t* scales, size_t* zeros) {
    ST_OK(check_shape(n, k, group));
    const size_t T = (n + 15) / 16, S = (k + 127) / 128, Q = (k + group - 1) / group;
    if (codes) *codes = T * S * 1024;
    if (scales) *scales = T * Q * 32;
    if (zeros) *zeros = T * Q * 16;
    return KV_OK;
}

int w4_quantize(const w4_matrix* m, const void* w, int dtype, long long ldw, void* stream) {
    ST_OK(check_matrix(m, "matrix"));
    if (dtype != STEP_F16 && dtype != STEP_BF16)
        return sfail(KV_ERR_INVAL, "weights to quantise are STEP_F16 or STEP_BF16, not %d", dtype);
    if (!w || !aligned(w, 2)) return sfail(KV_ERR_INVAL, "weights NULL or unaligned");
    if (ldw < m->k || ldw > (1ll << 40)) return sfail(KV_ERR_INVAL, "rows %lld apart for %d inputs", ldw, m->k);
    DeviceGuard g(m->device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", m->device);
    return launched(launch_w4_quantize(*m, w, dtype, ldw, static_cast<cudaStream_t>(stream)), "w4_quantize");
}

int w4_dequantize(const w4_matrix* m, float* out, long long ldo, void* stream) {
    ST_OK(check_matrix(m, "matrix"));
    if (!out || !aligned(out, 4)) return sfail(KV_ERR_INVAL, "out NULL or unaligned");
    if (ldo < m->k || ldo > (1ll << 40)) return sfail(KV_ERR_INVAL, "rows %lld apart for %d inputs", ldo, m->k);
    DeviceGuard g(m->device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", m->device);
    return launched(launch_w4_dequantize(*m, out, ldo, static_cast<cudaStream_t>(stream)), "w4_dequantize");
}

int w4_linear(const w4_matrix* w, const void* x, int x_dtype, int m, long long ldx, const float* bias,
              const void* residual, long long ldr, void* out, int out_dtype, long long ldo, void* work, void* stream) {
    ST_OK(check_matrix(w, "matrix"));
    ST_OK(check_rows(*w, x, x_dtype, m, ldx, out, out_dtype, ldo));
    ST_OK(check_work(*w, x, x_dtype, m, ldx, out, out_dtype, ldo, 0, work));
    if (!aligned(bias, 4)) return sfail(KV_ERR_INVAL, "bias is not aligned to its element");
    if (residual) {
        if (ldr < w->n || ldr > (1ll << 40)) return sfail(KV_ERR_INVAL, "residual rows %lld apart for %d outputs", ldr, w->n);
        if (!aligned(residual, esize(out_dtype))) return sfail(KV_ERR_INVAL, "residual is not aligned to its element");
        const size_t es = esize(out_dtype);
        if (!(residual == out && ldr == ldo) && Range(residual, m, w->n, ldr, es).meets(Range(out, m, w->n, ldo, es)))
            return sfail(KV_ERR_INVAL, "residual overlaps out without being out");
    }
    if (m == 0) return KV_OK;
    DeviceGuard g(w->device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", w->device);
    W4Args a;
    a.set_matrix(0, *w);
    set_x(a, x, x_dtype, m, ldx);
    a.work = work;
    a.mode = W4_LINEAR;
    a.bias = bias;
    a.residual = residual;
    a.ldr = ldr;
    a.out = out;
    a.out_dtype = out_dtype;
    a.ldo = ldo;
    return launched(launch_w4(a, w->group, x_dtype != STEP_F16, 1, static_cast<cudaStream_t>(stream)), "w4_linear");
}

int w4_gated(const w4_matrix* gate, const w4_matrix* up, const void* x, int x_dtype, int m, long long ldx, void* out,
             int out_dtype, long long ldo, void* work, void* stream) {
    ST_OK(check_matrix(gate, "gate matrix"));
    ST_OK(check_matrix(up, "up matrix"));
    if (gate->n != up->n || gate->k != up->k || gate->group != up->group || gate->device != up->device ||
        !gate->zeros != !up->zeros)
        return sfail(KV_ERR_INVAL, "gate and up differ in shape, group, device or zero points");
    ST_OK(check_rows(*gate, x, x_dtype, m, ldx, out, out_dtype, ldo));
    ST_OK(check_work(*gate, x, x_dtype, m, ldx, out, out_dtype, ldo, 1, work));
    if (m == 0) return KV_OK;
    DeviceGuard g(gate->device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", gate->device);
    W4Args a;
    a.set_matrix(0, *gate);
    a.set_matrix(1, *up);
    set_x(a, x, x_dtype, m, ldx);
    a.work = work;
    a.mode = W4_GATED;
    a.out = out;
    a.out_dtype = out_dtype;
    a.ldo = ldo;
    return launched(launch_w4(a, gate->group, x_dtype != STEP_F16, 2, static_cast<cudaStream_t>(stream)), "w4_gated");
}

int w4_work_bytes(int n, int k, int group, int x_dtype, int m, int gated, size_t* bytes) {
    ST_OK(check_shape(n, k, group));
    ST_OK(check_dtype(x_dtype, "x"));
    if (m < 0 || m > kMaxRows || !bytes) return sfail(KV_ERR_INVAL, "%d rows, or NULL bytes", m);
    *bytes = work_bytes(n, k, group, x_dtype, m, gated);
    return KV_OK;
}

int step_ops_status(int device, int* status) {
    if (!status || device < 0) return sfail(KV_ERR_INVAL, "NULL status or no device");
    DeviceGuard g(device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", device);
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = step_status(status);
    return launched(e, "step_ops_status");
}

int step_ops_wait_limit(long long clocks) {
    set_wait_limit(clocks);
    return KV_OK;
}

int logits_adjust(const logits_call* c, void* stream) {
    if (!c) return sfail(KV_ERR_INVAL, "NULL call");
    ST_OK(check_dtype(c->dtype, "logits"));
    if (c->rows < 0 || c->vocab <= 0 || c->vocab > kMaxDim)
        return sfail(KV_ERR_INVAL, "%d rows of %d logits", c->rows, c->vocab);
    if (c->rows > 65535) return sfail(KV_ERR_RANGE, "%d rows in one call (at most 65535)", c->rows);
    if (c->rows == 0) return KV_OK;
    if (!c->logits || !c->out) return sfail(KV_ERR_INVAL, "NULL logits or out");
    if (c->ld_logits < c->vocab || c->ld_out < c->vocab || c->ld_logits > (1ll << 40) || c->ld_out > (1ll << 40))
        return sfail(KV_ERR_INVAL, "rows %lld / %lld apart for %d logits", c->ld_logits, c->ld_out, c->vocab);
    const size_t es = esize(c->dtype);
    if (!aligned(c->logits, es) || !aligned(c->out, es)) return sfail(KV_ERR_INVAL, "logits or out not aligned to its element");
    if (!(c->logits == c->out && c->ld_logits == c->ld_out) &&
        Range(c->logits, c->rows, c->vocab, c->ld_logits, es).meets(Range(c->out, c->rows, c->vocab, c->ld_out, es)))
        return sfail(KV_ERR_INVAL, "out overlaps logits without being logits");
    if (c->hist && (!c->hist_off || c->hist_n < 0)) return sfail(KV_ERR_INVAL, "a history needs hist_off and hist_n");
    if (c->bias_ids && (!c->bias_off || !c->bias || c->bias_n < 0))
        return sfail(KV_ERR_INVAL, "a bias list needs bias, bias_off and bias_n");
    if (c->mask && c->ld_mask < ((long long)c->vocab + 31) / 32)
        return sfail(KV_ERR_INVAL, "mask rows of %lld words for %d logits", c->ld_mask, c->vocab);
    const void* words[] = {c->pick, c->hist, c->hist_off, c->gen_from, c->repetition, c->presence, c->frequency,
                           c->bias_ids, c->bias, c->bias_off, c->mask};
    for (const void* p : words)
        if (!aligned(p, 4)) return sfail(KV_ERR_INVAL, "an array of 4-byte values is not aligned");
    if (c->device < 0) return sfail(KV_ERR_INVAL, "no device");
    DeviceGuard g(c->device);
    if (!g.ok) return sfail(KV_ERR_INVAL, "no CUDA device %d", c->device);
    return launched(launch_logits(*c, static_cast<cudaStream_t>(stream)), "logits_adjust");
}

}  // extern "C"
