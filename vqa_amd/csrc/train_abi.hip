// C entry points of the softmax read-out and of the orthogonalised updates (include/vqa_hip.h): argument checks, the
// calling thread's device kept, nothing thrown across the boundary.
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <new>

#include "vqa_core.h"

using namespace vqa;

namespace {

struct DeviceScope {   // the call's device is current while it queues work; the caller's comes back
    int before = -1, device = -1;
    int enter(int d) {
        static const int count = [] { int n = 0; return hipGetDeviceCount(&n) == hipSuccess ? n : 0; }();
        if (d < 0 || d >= count) VQA_FAIL(VQA_ENODEVICE, "device %d out of range (%d visible)", d, count);
        VQA_HIP(hipGetDevice(&before));
        device = d;
        if (before != d) VQA_HIP(hipSetDevice(d));
        return VQA_OK;
    }
    ~DeviceScope() {
        if (before >= 0 && before != device) (void)hipSetDevice(before);
    }
};

struct Buf {   // device memory of a host-pointer call
    void* p = nullptr;
    ~Buf() { if (p) (void)hipFree(p); }
    int alloc(size_t bytes) {
        hipError_t e = hipMalloc(&p, std::max<size_t>(bytes, 16));
        if (e != hipSuccess) VQA_FAIL(VQA_ENOMEM, "hipMalloc(%zu) failed: %s", bytes, hipGetErrorString(e));
        return VQA_OK;
    }
    int upload(const void* src, size_t bytes, hipStream_t s) {
        if (!src) return VQA_OK;
        int rc = alloc(bytes);
        if (rc) return rc;
        VQA_HIP(hipMemcpyAsync(p, src, bytes, hipMemcpyHostToDevice, s));
        return VQA_OK;
    }
    int download(void* dst, size_t bytes, hipStream_t s) const {
        if (dst && bytes) VQA_HIP(hipMemcpyAsync(dst, p, bytes, hipMemcpyDeviceToHost, s));
        return VQA_OK;
    }
};
// what was queued has read the caller's memory and the buffers above before they go, also on the way out of an error
struct Waits {
    hipStream_t s = nullptr;
    bool on = false;
    ~Waits() { if (on) (void)hipStreamSynchronize(s); }
};

size_t size_of(int dtype) { return dtype == VQA_DTYPE_F64 ? 8 : dtype == VQA_DTYPE_F32 ? 4 : 2; }
size_t wide_of(int dtype) { return dtype == VQA_DTYPE_F64 ? 8 : 4; }
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na && nb && x < y + nb && y < x + na;
}

// kernels read and write whole values, and 16 bytes at once of a workspace
struct Aligned {
    const void* p;
    size_t to;
    const char* what;
};
int check_aligned(std::initializer_list<Aligned> all) {
    for (const Aligned& a : all)
        if ((uintptr_t)a.p % a.to) VQA_FAIL(VQA_EINVAL, "%s is not aligned to %zu bytes", a.what, a.to);
    return VQA_OK;
}
constexpr size_t kWorkspaceAlign = 16;

int check_dtype(int dtype) {
    if (dtype < 0 || dtype > 3) VQA_FAIL(VQA_EINVAL, "dtype must be one of VQA_DTYPE_* (got %d)", dtype);
    return VQA_OK;
}

// rows of scores; *bytes: from the first element to the last
int check_rows(int dtype, const void* z, int64_t rows, int64_t width, int64_t stride, const char* what, size_t* bytes) {
    if (rows < 0 || rows > ((int64_t)1 << 40)) VQA_FAIL(VQA_EINVAL, "rows must be in [0, 2^40] (got %lld)", (long long)rows);
    if (width < 1 || width > 0x7fffffff) VQA_FAIL(VQA_EINVAL, "width must be in [1, 2^31 - 1] (got %lld)", (long long)width);
    if (stride < width || stride > ((int64_t)1 << 40))
        VQA_FAIL(VQA_EINVAL, "the row stride of %s must be in [width, 2^40] (got %lld)", what, (long long)stride);
    if (rows > 0 && !z) VQA_FAIL(VQA_EINVAL, "%s is NULL", what);
    if (rows > 0 && rows > ((int64_t)1 << 58) / stride) VQA_FAIL(VQA_EINVAL, "%s is too large", what);
    if ((uintptr_t)z % size_of(dtype)) VQA_FAIL(VQA_EINVAL, "%s is not aligned to its type", what);
    *bytes = rows > 0 ? ((size_t)(rows - 1) * stride + width) * size_of(dtype) : 0;
    return VQA_OK;
}

int check_scale(double scale) {
    if (!(scale > 0.0) || !isfinite(scale) || scale > 1e30 || scale < 1e-30)
        VQA_FAIL(VQA_EINVAL, "scale must be in [1e-30, 1e30] (got %g)", scale);
    return VQA_OK;
}

struct Score {
    int dtype;
    const void* z;
    int64_t rows, width, stride;
    double scale;
    const int32_t* targets;
    int top_k;
    void *log_prob, *entropy, *top_log_prob;
    int32_t* top_index;
    size_t bytes;

    int check() {
        int rc = check_dtype(dtype);
        if (rc) return rc;
        if ((rc = check_rows(dtype, z, rows, width, stride, "scores", &bytes))) return rc;
        if ((rc = check_scale(scale))) return rc;
        if (top_k < 0 || top_k > std::min<int64_t>(64, width))
            VQA_FAIL(VQA_EINVAL, "top_k must be in [0, min(64, width)] (got %d)", top_k);
        if (rows == 0) return VQA_OK;
        if (top_k > 0 && (!top_log_prob || !top_index)) VQA_FAIL(VQA_EINVAL, "top_log_prob and top_index must not be NULL with top_k > 0");
        if (log_prob && !targets) VQA_FAIL(VQA_EINVAL, "log_prob needs the targets");
        return VQA_OK;
    }
    int check_aligned_to_types() const {     // device pointers
        const size_t w = wide_of(dtype);
        return check_aligned({ { targets, 4, "targets" }, { log_prob, w, "log_prob" }, { entropy, w, "entropy" },
                               { top_k ? top_log_prob : nullptr, w, "top_log_prob" }, { top_k ? top_index : nullptr, 4, "top_index" } });
    }
};

struct Loss {
    int dtype;
    const void* z;
    int64_t rows, width, stride;
    double scale;
    const int32_t* targets;
    const void *dlog_prob, *dentropy;
    void *log_prob, *entropy, *dz;
    int64_t dz_stride;
    size_t bytes, dz_bytes;

    // rows of one array, the scores in some of its columns and their gradient in others
    bool side_by_side() const {
        if (stride != dz_stride) return false;
        const int64_t d = ((int64_t)((intptr_t)dz - (intptr_t)z) / (int64_t)size_of(dtype) % stride + stride) % stride;
        return d >= width && stride - d >= width;
    }

    int check() {
        int rc = check_dtype(dtype);
        if (rc) return rc;
        if ((rc = check_rows(dtype, z, rows, width, stride, "scores", &bytes))) return rc;
        if ((rc = check_rows(dtype, dz, rows, width, dz_stride, "dscores", &dz_bytes))) return rc;
        if ((rc = check_scale(scale))) return rc;
        if (rows == 0) return VQA_OK;
        if ((log_prob || dlog_prob) && !targets) VQA_FAIL(VQA_EINVAL, "log_prob and dlog_prob need the targets");
        if (overlap(z, bytes, dz, dz_bytes) && !side_by_side()) VQA_FAIL(VQA_EINVAL, "dscores must not overlap the scores");
        return VQA_OK;
    }
    int check_aligned_to_types() const {     // device pointers
        const size_t w = wide_of(dtype);
        return check_aligned({ { targets, 4, "targets" }, { dlog_prob, w, "dlog_prob" }, { dentropy, w, "dentropy" },
                               { log_prob, w, "log_prob" }, { entropy, w, "entropy" } });
    }
};

// The singular values of X0 are at most 1; what the steps make of them, and of the polynomial of A that multiplies X.
int check_coefs(int steps, const double* k) {
    if (steps < 1 || steps > 100) VQA_FAIL(VQA_EINVAL, "steps must be in [1, 100] (got %d)", steps);
    if (!k) VQA_FAIL(VQA_EINVAL, "coefs is NULL");
    for (int i = 0; i < 3; ++i)
        if (!isfinite(k[i])) VQA_FAIL(VQA_EINVAL, "coefs must be finite");
    double most = 1.0;
    for (int s = 0; s < steps; ++s) {
        const double y = most * most, poly = fabs(k[1]) * y + fabs(k[2]) * y * y;
        if (poly > 32.0) VQA_FAIL(VQA_EUNSUPPORTED, "coefs (%g, %g, %g): the polynomial of X X^T reaches %g (at most 32)", k[0], k[1], k[2], poly);
        // the largest |p| on [0, most]: at its end, or where k0 + 3 k1 y + 5 k2 y^2 = 0 (y = the square)
        auto size = [&](double q) { return sqrt(q) * fabs(k[0] + q * (k[1] + q * k[2])); };
        double next = size(y);
        const double disc = 9 * k[1] * k[1] - 20 * k[0] * k[2];
        if (k[2] != 0.0 && disc >= 0.0) {
            for (double sign : { -1.0, 1.0 }) {
                const double q = (-3 * k[1] + sign * sqrt(disc)) / (10 * k[2]);
                if (q > 0.0 && q < y) next = std::max(next, size(q));
            }
        } else if (k[2] == 0.0 && k[1] != 0.0) {
            const double q = -k[0] / (3 * k[1]);
            if (q > 0.0 && q < y) next = std::max(next, size(q));
        }
        next = next * (1 + 1e-6) + 1e-6;      // (what roundings add)
        if (next > 4.0) VQA_FAIL(VQA_EUNSUPPORTED, "coefs (%g, %g, %g) carry a singular value to %g (at most 4)", k[0], k[1], k[2], next);
        most = next;
    }
    return VQA_OK;
}

int check_matrices(OrthoCall& q, const double* coefs, size_t* g_bytes) {
    int rc = check_dtype(q.dtype);
    if (rc) return rc;
    if (q.batch < 0 || q.batch > 65535) VQA_FAIL(VQA_EINVAL, "batch must be in [0, 65535] (got %d)", q.batch);
    if (q.rows < 1 || q.rows > 65536 || q.cols < 1 || q.cols > 65536)
        VQA_FAIL(VQA_EINVAL, "rows and cols must be in [1, 65536] (got %d x %d)", q.rows, q.cols);
    if (q.g_row_stride < q.cols || q.g_row_stride > ((int64_t)1 << 40))
        VQA_FAIL(VQA_EINVAL, "row_stride must be in [cols, 2^40] (got %lld)", (long long)q.g_row_stride);
    const int64_t one = (int64_t)(q.rows - 1) * q.g_row_stride + q.cols;
    if (q.batch > 1 && (q.g_batch_stride < one || q.g_batch_stride > ((int64_t)1 << 42)))
        VQA_FAIL(VQA_EINVAL, "batch_stride must be in [a matrix's extent, 2^42] (got %lld)", (long long)q.g_batch_stride);
    if (!(q.eps >= 1e-300) || !isfinite(q.eps)) VQA_FAIL(VQA_EINVAL, "eps must be at least 1e-300 and finite");
    if ((rc = check_coefs(q.steps, coefs))) return rc;
    if (ortho_in_pairs(q.dtype, q.rows, q.cols) && fabs(coefs[0]) < 1.0)
        VQA_FAIL(VQA_EUNSUPPORTED, "coefs (%g, %g, %g) shrink small singular values: of 32 and 16 bits, only matrices of up to 64 rows or columns take them", coefs[0], coefs[1], coefs[2]);
    std::copy(coefs, coefs + 3, q.coefs);
    *g_bytes = q.batch ? ((size_t)(q.batch - 1) * q.g_batch_stride + one) * size_of(q.dtype) : 0;
    if (q.batch && !q.g) VQA_FAIL(VQA_EINVAL, "g is NULL");
    if ((uintptr_t)q.g % size_of(q.dtype)) VQA_FAIL(VQA_EINVAL, "g is not aligned to its type");
    return VQA_OK;
}

size_t dense(const OrthoCall& q) { return (size_t)q.batch * q.rows * q.cols; }

int check_out(const OrthoCall& q, size_t g_bytes) {
    if (!q.batch) return VQA_OK;
    if (!q.out) VQA_FAIL(VQA_EINVAL, "out is NULL");
    const bool same = q.out == q.g && q.g_row_stride == q.cols && (q.batch == 1 || q.g_batch_stride == (int64_t)q.rows * q.cols);
    if (!same && overlap(q.g, g_bytes, q.out, dense(q) * size_of(q.dtype)))
        VQA_FAIL(VQA_EINVAL, "out must not overlap g, unless it is g and g is contiguous");
    return VQA_OK;
}

int check_step(const OrthoCall& q, size_t g_bytes) {
    if (!isfinite(q.lr) || !isfinite(q.mu) || !isfinite(q.weight_decay)) VQA_FAIL(VQA_EINVAL, "lr, mu and weight_decay must be finite");
    if (!q.batch) return VQA_OK;
    if (!q.weight || !q.momentum) VQA_FAIL(VQA_EINVAL, "weight and momentum must not be NULL");
    const size_t n = dense(q) * wide_of(q.dtype);
    if (overlap(q.weight, n, q.momentum, n) || overlap(q.weight, n, q.g, g_bytes) || overlap(q.momentum, n, q.g, g_bytes))
        VQA_FAIL(VQA_EINVAL, "weight, momentum and g must not overlap");
    return VQA_OK;
}

int queue_ortho(int device, void* stream, OrthoCall& q) {
    if (!q.batch) return VQA_OK;
    if (!q.workspace && ortho_workspace_bytes(q.dtype, q.batch, q.rows, q.cols)) VQA_FAIL(VQA_EINVAL, "workspace is NULL");
    int rc = check_aligned({ { q.out, size_of(q.dtype), "out" }, { q.weight, wide_of(q.dtype), "weight" }, { q.momentum, wide_of(q.dtype), "momentum" },
                             { q.workspace, kWorkspaceAlign, "workspace" } });
    if (rc) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    return ortho_launch((hipStream_t)stream, q);
}

}  // namespace

#define VQA_ENTRY try {
#define VQA_EXIT                                                                                 \
    }                                                                                            \
    catch (const std::bad_alloc&) { VQA_FAIL(VQA_ENOMEM, "out of host memory"); }                \
    catch (...) { VQA_FAIL(VQA_EINVAL, "unexpected host error"); }

extern "C" {

int64_t vqa_log_probs_workspace(int dtype, int64_t rows, int64_t width, int top_k) {
    if (dtype < 0 || dtype > 3 || rows < 0 || width < 1 || top_k < 0 || top_k > 64) return 0;
    return (int64_t)log_probs_workspace_bytes(dtype, rows, width, top_k);
}

int vqa_log_probs_dev(int device, void* stream, int dtype, const void* d_scores, int64_t rows, int64_t width, int64_t row_stride,
                      double scale, const int32_t* d_targets, int top_k, void* d_workspace, void* d_log_prob, void* d_entropy,
                      void* d_top_log_prob, int32_t* d_top_index) {
    VQA_ENTRY
    Score q = { dtype, d_scores, rows, width, row_stride, scale, d_targets, top_k, d_log_prob, d_entropy, d_top_log_prob, d_top_index, 0 };
    int rc = q.check();
    if (rc || rows == 0) return rc;
    if ((rc = q.check_aligned_to_types())) return rc;
    if (!d_workspace && log_probs_workspace_bytes(dtype, rows, width, top_k)) VQA_FAIL(VQA_EINVAL, "workspace is NULL");
    if ((rc = check_aligned({ { d_workspace, kWorkspaceAlign, "workspace" } }))) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    return log_probs_launch((hipStream_t)stream, dtype, d_scores, rows, width, row_stride, scale, d_targets, top_k, d_workspace,
                            d_log_prob, d_entropy, d_top_log_prob, d_top_index);
    VQA_EXIT
}

int vqa_log_probs(int device, int dtype, const void* scores, int64_t rows, int64_t width, int64_t row_stride, double scale,
                  const int32_t* targets, int top_k, void* log_prob, void* entropy, void* top_log_prob, int32_t* top_index) {
    VQA_ENTRY
    Score q = { dtype, scores, rows, width, row_stride, scale, targets, top_k, log_prob, entropy, top_log_prob, top_index, 0 };
    int rc = q.check();
    if (rc || rows == 0) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    const size_t w = wide_of(dtype), n = (size_t)rows;
    Buf z, t, lp, en, tl, ti, ws;
    Waits wait;
    if ((rc = library_stream(device, &wait.s))) return rc;
    wait.on = true;
    if ((rc = z.upload(scores, q.bytes, wait.s)) || (rc = t.upload(targets, n * 4, wait.s))) return rc;
    if ((log_prob && (rc = lp.alloc(n * w))) || (entropy && (rc = en.alloc(n * w)))) return rc;
    if (top_k && ((rc = tl.alloc(n * top_k * w)) || (rc = ti.alloc(n * top_k * 4)))) return rc;
    if ((rc = ws.alloc(log_probs_workspace_bytes(dtype, rows, width, top_k)))) return rc;
    if ((rc = log_probs_launch(wait.s, dtype, z.p, rows, width, row_stride, scale, (const int32_t*)t.p, top_k, ws.p, lp.p, en.p, tl.p,
                               (int32_t*)ti.p)))
        return rc;
    if ((rc = lp.download(log_prob, n * w, wait.s)) || (rc = en.download(entropy, n * w, wait.s))) return rc;
    if (top_k && ((rc = tl.download(top_log_prob, n * top_k * w, wait.s)) || (rc = ti.download(top_index, n * top_k * 4, wait.s)))) return rc;
    VQA_HIP(hipStreamSynchronize(wait.s));
    return VQA_OK;
    VQA_EXIT
}

int vqa_log_probs_grad_dev(int device, void* stream, int dtype, const void* d_scores, int64_t rows, int64_t width,
                           int64_t row_stride, double scale, const int32_t* d_targets, const void* d_dlog_prob,
                           const void* d_dentropy, void* d_workspace, void* d_log_prob, void* d_entropy, void* d_dscores,
                           int64_t dscores_row_stride) {
    VQA_ENTRY
    Loss q = { dtype, d_scores, rows, width, row_stride, scale, d_targets, d_dlog_prob, d_dentropy, d_log_prob, d_entropy,
               d_dscores, dscores_row_stride, 0, 0 };
    int rc = q.check();
    if (rc || rows == 0) return rc;
    if ((rc = q.check_aligned_to_types())) return rc;
    if (!d_workspace && log_probs_workspace_bytes(dtype, rows, width, 0)) VQA_FAIL(VQA_EINVAL, "workspace is NULL");
    if ((rc = check_aligned({ { d_workspace, kWorkspaceAlign, "workspace" } }))) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    return log_probs_grad_launch((hipStream_t)stream, dtype, d_scores, rows, width, row_stride, scale, d_targets, d_dlog_prob,
                                 d_dentropy, d_workspace, d_log_prob, d_entropy, d_dscores, dscores_row_stride);
    VQA_EXIT
}

int vqa_log_probs_grad(int device, int dtype, const void* scores, int64_t rows, int64_t width, int64_t row_stride, double scale,
                       const int32_t* targets, const void* dlog_prob, const void* dentropy, void* log_prob, void* entropy,
                       void* dscores, int64_t dscores_row_stride) {
    VQA_ENTRY
    Loss q = { dtype, scores, rows, width, row_stride, scale, targets, dlog_prob, dentropy, log_prob, entropy, dscores,
               dscores_row_stride, 0, 0 };
    int rc = q.check();
    if (rc || rows == 0) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    const size_t w = wide_of(dtype), n = (size_t)rows;
    Buf z, t, g, h, lp, en, dz, ws;
    Waits wait;
    if ((rc = library_stream(device, &wait.s))) return rc;
    wait.on = true;
    if ((rc = z.upload(scores, q.bytes, wait.s)) || (rc = t.upload(targets, n * 4, wait.s))) return rc;
    if ((rc = g.upload(dlog_prob, n * w, wait.s)) || (rc = h.upload(dentropy, n * w, wait.s))) return rc;
    if ((log_prob && (rc = lp.alloc(n * w))) || (entropy && (rc = en.alloc(n * w)))) return rc;
    if ((rc = ws.alloc(log_probs_workspace_bytes(dtype, rows, width, 0)))) return rc;
    if ((rc = dz.upload(dscores, q.dz_bytes, wait.s))) return rc;   // what lies between the rows comes back as it was
    if ((rc = log_probs_grad_launch(wait.s, dtype, z.p, rows, width, row_stride, scale, (const int32_t*)t.p, g.p, h.p, ws.p, lp.p,
                                    en.p, dz.p, dscores_row_stride)))
        return rc;
    if ((rc = lp.download(log_prob, n * w, wait.s)) || (rc = en.download(entropy, n * w, wait.s))) return rc;
    if ((rc = dz.download(dscores, q.dz_bytes, wait.s))) return rc;
    VQA_HIP(hipStreamSynchronize(wait.s));
    return VQA_OK;
    VQA_EXIT
}

int64_t vqa_psr_chain_workspace(int64_t n_samples, int n_params) {
    if (n_samples < 0 || n_samples > ((int64_t)1 << 22) || n_params < 1) return 0;
    return (int64_t)psr_chain_workspace_bytes(n_samples, n_params);
}

int vqa_psr_chain_dev(int device, void* stream, const double* d_expect, int64_t n_samples, int n_params, int n_obs, double factor,
                      const double* d_dexpect, double* d_workspace, double* d_out) {
    VQA_ENTRY
    if (n_samples < 0 || n_samples > ((int64_t)1 << 22)) VQA_FAIL(VQA_EINVAL, "n_samples must be in [0, 2^22] (got %lld)", (long long)n_samples);
    if (n_params < 0 || n_params > (1 << 20) || n_obs < 1) VQA_FAIL(VQA_EINVAL, "n_params must be in [0, 2^20] and n_obs >= 1");
    if (n_params == 0) return VQA_OK;
    if (!d_out) VQA_FAIL(VQA_EINVAL, "out is NULL");
    if (n_samples > 0 && (!d_expect || !d_dexpect || !d_workspace)) VQA_FAIL(VQA_EINVAL, "expect, dexpect and workspace must not be NULL");
    int rc = check_aligned({ { d_expect, 8, "expect" }, { d_dexpect, 8, "dexpect" }, { d_workspace, 8, "workspace" }, { d_out, 8, "out" } });
    if (rc) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    return psr_chain_launch((hipStream_t)stream, d_expect, n_samples, n_params, n_obs, factor, d_dexpect, d_workspace, d_out);
    VQA_EXIT
}

int64_t vqa_orthogonalize_workspace(int dtype, int batch, int rows, int cols) {
    if (dtype < 0 || dtype > 3 || batch < 0 || rows < 1 || cols < 1 || rows > 65536 || cols > 65536) return 0;
    return (int64_t)ortho_workspace_bytes(dtype, batch, rows, cols);
}

int vqa_orthogonalize_dev(int device, void* stream, int dtype, const void* d_g, int batch, int rows, int cols, int64_t row_stride,
                          int64_t batch_stride, int steps, const double* coefs, double eps, void* d_workspace, void* d_out) {
    VQA_ENTRY
    OrthoCall q = {};
    q.dtype = dtype; q.g = d_g; q.g_row_stride = row_stride; q.g_batch_stride = batch_stride;
    q.batch = batch; q.rows = rows; q.cols = cols; q.steps = steps; q.eps = eps; q.workspace = d_workspace; q.out = d_out;
    size_t bytes;
    int rc = check_matrices(q, coefs, &bytes);
    if (rc || (rc = check_out(q, bytes))) return rc;
    return queue_ortho(device, stream, q);
    VQA_EXIT
}

int vqa_orthogonalize(int device, int dtype, const void* g, int batch, int rows, int cols, int64_t row_stride, int64_t batch_stride,
                      int steps, const double* coefs, double eps, void* out) {
    VQA_ENTRY
    OrthoCall q = {};
    q.dtype = dtype; q.g = g; q.g_row_stride = row_stride; q.g_batch_stride = batch_stride;
    q.batch = batch; q.rows = rows; q.cols = cols; q.steps = steps; q.eps = eps; q.out = out;
    size_t bytes;
    int rc = check_matrices(q, coefs, &bytes);
    if (rc || (rc = check_out(q, bytes)) || !batch) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    const size_t n = dense(q) * size_of(dtype);
    Buf dg, dout, ws;
    Waits wait;
    if ((rc = library_stream(device, &wait.s))) return rc;
    wait.on = true;
    if ((rc = dg.upload(g, bytes, wait.s)) || (rc = dout.alloc(n)) || (rc = ws.alloc(ortho_workspace_bytes(dtype, batch, rows, cols)))) return rc;
    q.g = dg.p; q.out = dout.p; q.workspace = ws.p;
    if ((rc = queue_ortho(device, wait.s, q)) || (rc = dout.download(out, n, wait.s))) return rc;
    VQA_HIP(hipStreamSynchronize(wait.s));
    return VQA_OK;
    VQA_EXIT
}

int vqa_muon_step_dev(int device, void* stream, int dtype, void* d_weight, const void* d_g, void* d_momentum, int batch, int rows,
                      int cols, int64_t row_stride, int64_t batch_stride, double lr, double mu, double weight_decay, int nesterov,
                      int steps, const double* coefs, double eps, void* d_workspace) {
    VQA_ENTRY
    OrthoCall q = {};
    q.dtype = dtype; q.g = d_g; q.g_row_stride = row_stride; q.g_batch_stride = batch_stride;
    q.batch = batch; q.rows = rows; q.cols = cols; q.steps = steps; q.eps = eps; q.workspace = d_workspace;
    q.weight = d_weight; q.momentum = d_momentum; q.lr = lr; q.mu = mu; q.weight_decay = weight_decay; q.nesterov = nesterov != 0;
    size_t bytes;
    int rc = check_matrices(q, coefs, &bytes);
    if (rc || (rc = check_step(q, bytes))) return rc;
    return queue_ortho(device, stream, q);
    VQA_EXIT
}

int vqa_muon_step(int device, int dtype, void* weight, const void* g, void* momentum, int batch, int rows, int cols,
                  int64_t row_stride, int64_t batch_stride, double lr, double mu, double weight_decay, int nesterov, int steps,
                  const double* coefs, double eps) {
    VQA_ENTRY
    OrthoCall q = {};
    q.dtype = dtype; q.g = g; q.g_row_stride = row_stride; q.g_batch_stride = batch_stride;
    q.batch = batch; q.rows = rows; q.cols = cols; q.steps = steps; q.eps = eps;
    q.weight = weight; q.momentum = momentum; q.lr = lr; q.mu = mu; q.weight_decay = weight_decay; q.nesterov = nesterov != 0;
    size_t bytes;
    int rc = check_matrices(q, coefs, &bytes);
    if (rc || (rc = check_step(q, bytes)) || !batch) return rc;
    DeviceScope scope;
    if ((rc = scope.enter(device))) return rc;
    const size_t n = dense(q) * wide_of(dtype);
    Buf dg, dw, dm, ws;
    Waits wait;
    if ((rc = library_stream(device, &wait.s))) return rc;
    wait.on = true;
    if ((rc = dg.upload(g, bytes, wait.s)) || (rc = dw.upload(weight, n, wait.s)) || (rc = dm.upload(momentum, n, wait.s)) ||
        (rc = ws.alloc(ortho_workspace_bytes(dtype, batch, rows, cols))))
        return rc;
    q.g = dg.p; q.weight = dw.p; q.momentum = dm.p; q.workspace = ws.p;
    if ((rc = queue_ortho(device, wait.s, q)) || (rc = dw.download(weight, n, wait.s)) || (rc = dm.download(momentum, n, wait.s))) return rc;
    VQA_HIP(hipStreamSynchronize(wait.s));
    return VQA_OK;
    VQA_EXIT
}

}  // extern "C"
