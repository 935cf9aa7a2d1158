// Host side of the microscaled entry points of include/turboloader_b200.h: argument checks, then one
// enqueue.  Nothing here allocates or synchronises.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/turboloader_b200.h"
#include "mx_params.h"

namespace tlb {
int report(int code, const char* message);  // capi.cu: sets tlb_last_error() and returns code
}

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return tlb::report(code, buf);
}

int cuda_fail(int e, const char* what) {
    return fail(TLB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(static_cast<cudaError_t>(e)));
}

// The kernels exist for sm_100a only, and the current device has to be one.
int need_device() {
    int dev = 0, major = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TLB_ERR_NO_DEVICE, "no CUDA device: %s", cudaGetErrorString(e));
    }
    if (major != 10) return fail(TLB_ERR_NO_DEVICE, "the current device is not an sm_100 GPU");
    return TLB_OK;
}

bool misaligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

int check_dtype(int dtype, const char* what) {
    if (dtype != TLB_F32 && dtype != TLB_BF16 && dtype != TLB_F16) return fail(TLB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
    return TLB_OK;
}

int check_rows(const tlb_mx_rows* q, const char* what) {
    if (!q) return fail(TLB_ERR_INVALID_ARG, "%s is NULL", what);
    if (q->format < TLB_MX_NVFP4 || q->format > TLB_MX_MXFP8) return fail(TLB_ERR_INVALID_ARG, "%s: unknown format %d", what, q->format);
    if (q->rows < 0) return fail(TLB_ERR_INVALID_ARG, "%s: %lld rows", what, static_cast<long long>(q->rows));
    if (q->cols <= 0 || q->cols > TLB_MX_MAX_COLS) return fail(TLB_ERR_INVALID_ARG, "%s: cols = %d outside [1, %d]", what, q->cols, TLB_MX_MAX_COLS);
    if (q->rows > TLB_MX_MAX_ROWS) return fail(TLB_ERR_TOO_LARGE, "%s: %lld rows exceed %lld", what, static_cast<long long>(q->rows), static_cast<long long>(TLB_MX_MAX_ROWS));
    if (!(q->scale > 0.0f) || !std::isfinite(q->scale)) return fail(TLB_ERR_INVALID_ARG, "%s: scale must be positive and finite", what);
    if (q->rows > 0 && (!q->codes || !q->scales)) return fail(TLB_ERR_INVALID_ARG, "%s: codes and scales must be non-NULL", what);
    if (misaligned(q->codes, 16) || misaligned(q->scales, 4) || misaligned(q->scale_dev, 4))
        return fail(TLB_ERR_INVALID_ARG, "%s: codes need 16-byte, scales and scale_dev 4-byte alignment", what);
    return TLB_OK;
}

tlb::MxRows rows_of(const tlb_mx_rows& q) {
    return {q.codes, q.scales, q.rows, q.cols, q.format, q.scale, q.scale_dev};
}

int check_cache(const tlb_mx_cache* c) {
    if (!c) return fail(TLB_ERR_INVALID_ARG, "cache is NULL");
    if (int rc = check_rows(&c->rows, "cache")) return rc;
    if (c->tokens <= 0) return fail(TLB_ERR_INVALID_ARG, "cache: tokens = %d must be positive", c->tokens);
    if (c->rows.rows % c->tokens) return fail(TLB_ERR_INVALID_ARG, "cache: %lld rows are no whole number of samples of %d", static_cast<long long>(c->rows.rows), c->tokens);
    if (misaligned(c->lengths, 4) || misaligned(c->owner, 4) || misaligned(c->status, 4))
        return fail(TLB_ERR_INVALID_ARG, "cache: lengths, owner and status need 4-byte alignment");
    return TLB_OK;
}

int check_samples(const tlb_mx_cache& c, const int64_t* index, int64_t n) {
    const int64_t slots = c.rows.rows / c.tokens;
    if (n < 0) return fail(TLB_ERR_INVALID_ARG, "n = %lld is negative", static_cast<long long>(n));
    if (n > TLB_MX_MAX_ROWS / c.tokens) return fail(TLB_ERR_TOO_LARGE, "%lld samples of %d rows exceed %lld rows", static_cast<long long>(n), c.tokens, static_cast<long long>(TLB_MX_MAX_ROWS));
    if (!index && n > slots) return fail(TLB_ERR_BAD_INDEX, "n = %lld exceeds the cache's %lld samples without an index", static_cast<long long>(n), static_cast<long long>(slots));
    if (misaligned(index, 8)) return fail(TLB_ERR_INVALID_ARG, "index needs 8-byte alignment");
    return TLB_OK;
}

tlb::MxMove move_of(const tlb_mx_cache& c, const int64_t* index, int64_t n) {
    tlb::MxMove p{};
    p.q = rows_of(c.rows);
    p.slots = c.rows.rows / c.tokens;
    p.tokens = c.tokens;
    p.n = n;
    p.index = reinterpret_cast<const long long*>(index);
    p.cache_lengths = c.lengths;
    p.owner = c.owner;
    p.status = c.status;
    return p;
}

int check_product(const tlb_mx_rows* a, const tlb_mx_rows* b, int out_dtype) {
    if (int rc = check_rows(a, "a")) return rc;
    if (int rc = check_rows(b, "b")) return rc;
    if (a->format != b->format) return fail(TLB_ERR_INVALID_ARG, "a and b must have the same format");
    if (a->cols != b->cols) return fail(TLB_ERR_INVALID_ARG, "a has %d columns, b has %d", a->cols, b->cols);
    if (!std::isnormal(a->scale * b->scale)) return fail(TLB_ERR_INVALID_ARG, "the product of the tensor scales, %g and %g, leaves fp32's range", a->scale, b->scale);
    if (b->rows > TLB_MX_MAX_COLS) return fail(TLB_ERR_TOO_LARGE, "b: %lld rows exceed %d", static_cast<long long>(b->rows), TLB_MX_MAX_COLS);
    return check_dtype(out_dtype, "out");
}

tlb::MxProduct product_of(const tlb_mx_rows& a, const tlb_mx_rows& b, int out_dtype) {
    tlb::MxProduct p{};
    p.a = rows_of(a);
    p.b = rows_of(b);
    p.out_dtype = out_dtype;
    return p;
}

int check_quantize(const tlb_mx_rows* q, const void* x, int x_dtype, int64_t x_pitch) {
    if (int rc = check_rows(q, "q")) return rc;
    if (int rc = check_dtype(x_dtype, "x")) return rc;
    if (q->rows == 0) return TLB_OK;
    if (!x) return fail(TLB_ERR_INVALID_ARG, "x is NULL");
    if (q->rows > 1 && x_pitch < q->cols) return fail(TLB_ERR_INVALID_ARG, "x: row pitch %lld is less than %d columns", static_cast<long long>(x_pitch), q->cols);
    if (misaligned(x, x_dtype == TLB_F32 ? 4 : 2)) return fail(TLB_ERR_INVALID_ARG, "x is not aligned to its type");
    return TLB_OK;
}

int quantize(const tlb_mx_rows& q, const void* x, int x_dtype, int64_t x_pitch, void* stream) {
    tlb::MxMove p{};
    p.q = rows_of(q);
    p.slots = p.n = q.rows;
    p.tokens = 1;
    p.in = x;
    p.dtype = x_dtype;
    p.row_pitch = 0;
    p.sample_pitch = x_pitch;
    if (int e = tlb::launch_mx_write(p, stream)) return cuda_fail(e, "mx_quantize");
    return TLB_OK;
}

int check_matmul(tlb::MxProduct& p, const tlb_mx_rows* a, const tlb_mx_rows* b, void* out, int out_dtype, void* workspace, int64_t workspace_bytes) {
    if (int rc = check_product(a, b, out_dtype)) return rc;
    if (a->rows == 0 || b->rows == 0) return TLB_OK;
    if (!out) return fail(TLB_ERR_INVALID_ARG, "out is NULL");
    if (misaligned(out, 16)) return fail(TLB_ERR_INVALID_ARG, "out needs 16-byte alignment");
    p = product_of(*a, *b, out_dtype);
    const int64_t need = static_cast<int64_t>(tlb::mx_matmul_workspace(p));
    if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 256)))
        return fail(TLB_ERR_INVALID_ARG, "workspace of %lld bytes (256-byte aligned) is needed", static_cast<long long>(need));
    p.out = out;
    p.workspace = workspace;
    return TLB_OK;
}

// Fills p but for its pointers to g and the workspace; the results' only say which are wanted.
int check_grad(tlb::MxGrad& p, int g_dtype, int64_t m, int64_t n, const tlb_mx_rows* a, const tlb_mx_rows* b, const void* grad_a, int32_t grad_a_dtype,
               const void* grad_b, int32_t grad_b_dtype) {
    if (int rc = check_dtype(g_dtype, "g")) return rc;
    if (m < 0 || n < 0) return fail(TLB_ERR_INVALID_ARG, "g is %lld x %lld", static_cast<long long>(m), static_cast<long long>(n));
    if (m > TLB_MX_MAX_ROWS / 2 || n > TLB_MX_MAX_COLS) return fail(TLB_ERR_TOO_LARGE, "g: %lld x %lld is too large", static_cast<long long>(m), static_cast<long long>(n));
    if (!grad_a && !grad_b) return fail(TLB_ERR_INVALID_ARG, "no gradient is asked for");
    if (grad_b) {
        if (int rc = check_rows(a, "a")) return rc;
        if (int rc = check_dtype(grad_b_dtype, "grad_b")) return rc;
        if (a->rows != m) return fail(TLB_ERR_INVALID_ARG, "a has %lld rows, g has %lld", static_cast<long long>(a->rows), static_cast<long long>(m));
        p.a = rows_of(*a);
    }
    if (grad_a) {
        if (int rc = check_rows(b, "b")) return rc;
        if (int rc = check_dtype(grad_a_dtype, "grad_a")) return rc;
        if (b->rows != n) return fail(TLB_ERR_INVALID_ARG, "b has %lld rows, g has %lld columns", static_cast<long long>(b->rows), static_cast<long long>(n));
        p.b = rows_of(*b);
    }
    if (grad_a && grad_b && (a->format != b->format || a->cols != b->cols)) return fail(TLB_ERR_INVALID_ARG, "a and b must have the same format and columns");
    p.g_dtype = g_dtype;
    p.m = m;
    p.n = static_cast<int>(n);
    p.grad_a = const_cast<void*>(grad_a);
    p.grad_b = const_cast<void*>(grad_b);
    p.grad_a_dtype = grad_a_dtype;
    p.grad_b_dtype = grad_b_dtype;
    return TLB_OK;
}

}  // namespace

extern "C" {

int64_t tlb_mx_code_pitch(int32_t format, int32_t cols) {
    if (format < TLB_MX_NVFP4 || format > TLB_MX_MXFP8 || cols <= 0 || cols > TLB_MX_MAX_COLS) return -1;
    return tlb::mx_code_pitch(format, cols);
}

int64_t tlb_mx_scale_pitch(int32_t format, int32_t cols) {
    if (format < TLB_MX_NVFP4 || format > TLB_MX_MXFP8 || cols <= 0 || cols > TLB_MX_MAX_COLS) return -1;
    return tlb::mx_scale_pitch(format, cols);
}

int tlb_mx_quantize(const tlb_mx_rows* q, const void* x, int32_t x_dtype, int64_t x_pitch, void* stream) {
    if (int rc = check_quantize(q, x, x_dtype, x_pitch)) return rc;
    if (q->rows == 0) return TLB_OK;
    if (int rc = need_device()) return rc;
    return quantize(*q, x, x_dtype, x_pitch, stream);
}

int tlb_mx_write(const tlb_mx_cache* cache, const int64_t* index, int64_t n, const void* x, int32_t x_dtype,
                 int64_t row_pitch, int64_t sample_pitch, const int32_t* lengths, void* stream) {
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_samples(*cache, index, n)) return rc;
    if (int rc = check_dtype(x_dtype, "x")) return rc;
    if (n == 0) return TLB_OK;
    if (!index) return fail(TLB_ERR_INVALID_ARG, "index is NULL");
    if (!x) return fail(TLB_ERR_INVALID_ARG, "x is NULL");
    if (n > TLB_MX_SCAN_SAMPLES && !cache->owner)
        return fail(TLB_ERR_INVALID_ARG, "cache: a write of more than %d samples needs owner", TLB_MX_SCAN_SAMPLES);
    if (lengths && !cache->lengths) return fail(TLB_ERR_INVALID_ARG, "lengths given for a cache without lengths");
    if ((cache->tokens > 1 && row_pitch < cache->rows.cols) || (n > 1 && sample_pitch < cache->rows.cols))
        return fail(TLB_ERR_INVALID_ARG, "x: pitches %lld, %lld are less than %d columns", static_cast<long long>(row_pitch), static_cast<long long>(sample_pitch), cache->rows.cols);
    if (misaligned(x, x_dtype == TLB_F32 ? 4 : 2) || misaligned(lengths, 4)) return fail(TLB_ERR_INVALID_ARG, "x or lengths is not aligned to its type");
    if (int rc = need_device()) return rc;
    tlb::MxMove p = move_of(*cache, index, n);
    p.in = x;
    p.dtype = x_dtype;
    p.row_pitch = row_pitch;
    p.sample_pitch = sample_pitch;
    p.lengths = lengths;
    if (int e = tlb::launch_mx_write(p, stream)) return cuda_fail(e, "mx_write");
    return TLB_OK;
}

int tlb_mx_read(const tlb_mx_cache* cache, const int64_t* index, int64_t n, void* out, int32_t out_dtype,
                int32_t* lengths_out, void* stream) {
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_samples(*cache, index, n)) return rc;
    if (int rc = check_dtype(out_dtype, "out")) return rc;
    if (n == 0) return TLB_OK;
    if (!out) return fail(TLB_ERR_INVALID_ARG, "out is NULL");
    if (misaligned(out, 16) || misaligned(lengths_out, 4)) return fail(TLB_ERR_INVALID_ARG, "out needs 16-byte, lengths_out 4-byte alignment");
    if (int rc = need_device()) return rc;
    tlb::MxMove p = move_of(*cache, index, n);
    p.out = out;
    p.dtype = out_dtype;
    p.lengths_out = lengths_out;
    if (int e = tlb::launch_mx_read(p, stream)) return cuda_fail(e, "mx_read");
    return TLB_OK;
}

int tlb_mx_read_codes(const tlb_mx_cache* cache, const int64_t* index, int64_t n, uint8_t* codes, uint8_t* scales,
                      int32_t* lengths_out, void* stream) {
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_samples(*cache, index, n)) return rc;
    if (n == 0) return TLB_OK;
    if (!codes || !scales) return fail(TLB_ERR_INVALID_ARG, "codes and scales must be non-NULL");
    if (misaligned(codes, 16) || misaligned(scales, 4) || misaligned(lengths_out, 4))
        return fail(TLB_ERR_INVALID_ARG, "codes need 16-byte, scales and lengths_out 4-byte alignment");
    if (int rc = need_device()) return rc;
    tlb::MxMove p = move_of(*cache, index, n);
    p.out_codes = codes;
    p.out_scales = scales;
    p.lengths_out = lengths_out;
    if (int e = tlb::launch_mx_read_codes(p, stream)) return cuda_fail(e, "mx_read_codes");
    return TLB_OK;
}

int64_t tlb_mx_matmul_workspace(const tlb_mx_rows* a, const tlb_mx_rows* b, int32_t out_dtype) {
    if (check_product(a, b, out_dtype)) return -1;
    return static_cast<int64_t>(tlb::mx_matmul_workspace(product_of(*a, *b, out_dtype)));
}

int tlb_mx_matmul(const tlb_mx_rows* a, const tlb_mx_rows* b, void* out, int32_t out_dtype, void* workspace,
                  int64_t workspace_bytes, void* stream) {
    tlb::MxProduct p{};
    if (int rc = check_matmul(p, a, b, out, out_dtype, workspace, workspace_bytes)) return rc;
    if (a->rows == 0 || b->rows == 0) return TLB_OK;
    if (int rc = need_device()) return rc;
    if (int e = tlb::launch_mx_matmul(p, stream)) return cuda_fail(e, "mx_matmul");
    return TLB_OK;
}

int tlb_mx_linear(const tlb_mx_rows* a, const void* x, int32_t x_dtype, int64_t x_pitch, const tlb_mx_rows* b, const void* w,
                  int32_t w_dtype, int64_t w_pitch, void* out, int32_t out_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    tlb::MxProduct p{};
    if (int rc = check_matmul(p, a, b, out, out_dtype, workspace, workspace_bytes)) return rc;
    if (x)
        if (int rc = check_quantize(a, x, x_dtype, x_pitch)) return rc;
    if (w)
        if (int rc = check_quantize(b, w, w_dtype, w_pitch)) return rc;
    if (a->rows == 0 && b->rows == 0) return TLB_OK;
    if (int rc = need_device()) return rc;
    if (x && a->rows > 0)
        if (int rc = quantize(*a, x, x_dtype, x_pitch, stream)) return rc;
    if (w && b->rows > 0)
        if (int rc = quantize(*b, w, w_dtype, w_pitch, stream)) return rc;
    if (a->rows == 0 || b->rows == 0) return TLB_OK;
    if (int e = tlb::launch_mx_matmul(p, stream)) return cuda_fail(e, "mx_linear");
    return TLB_OK;
}

int tlb_mx_incomplete(uint32_t* count) {
    if (!count) return fail(TLB_ERR_INVALID_ARG, "count is NULL");
    *count = 0;
    if (int rc = need_device()) return rc;
    if (int e = tlb::mx_gave_up(count)) return cuda_fail(e, "mx_incomplete");
    return TLB_OK;
}

int64_t tlb_mx_grad_workspace(int32_t g_dtype, int64_t m, int64_t n, const tlb_mx_rows* a, const tlb_mx_rows* b, const void* grad_a,
                              int32_t grad_a_dtype, const void* grad_b, int32_t grad_b_dtype) {
    tlb::MxGrad p{};
    if (check_grad(p, g_dtype, m, n, a, b, grad_a, grad_a_dtype, grad_b, grad_b_dtype)) return -1;
    return static_cast<int64_t>(tlb::mx_grad_workspace(p));
}

int tlb_mx_grad(const void* g, int32_t g_dtype, int64_t m, int64_t n, const tlb_mx_rows* a, const tlb_mx_rows* b, void* grad_a,
                int32_t grad_a_dtype, void* grad_b, int32_t grad_b_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    tlb::MxGrad p{};
    if (int rc = check_grad(p, g_dtype, m, n, a, b, grad_a, grad_a_dtype, grad_b, grad_b_dtype)) return rc;
    if (!g && m > 0 && n > 0) return fail(TLB_ERR_INVALID_ARG, "g is NULL");
    if (misaligned(grad_a, 16) || misaligned(grad_b, 16) || misaligned(g, 16)) return fail(TLB_ERR_INVALID_ARG, "g, grad_a and grad_b need 16-byte alignment");
    const int64_t need = static_cast<int64_t>(tlb::mx_grad_workspace(p));
    if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 256)))
        return fail(TLB_ERR_INVALID_ARG, "workspace of %lld bytes (256-byte aligned) is needed", static_cast<long long>(need));
    if ((!grad_a || m == 0) && (!grad_b || n == 0)) return TLB_OK;
    if (int rc = need_device()) return rc;
    p.g = g;
    p.workspace = workspace;
    if (int e = tlb::launch_mx_grad(p, stream)) return cuda_fail(e, "mx_grad");
    return TLB_OK;
}

}  // extern "C"
