/*
 * The training of linear layers and ReLU^2 MLPs from 8-bit checkpoints, a direction a call: the quantizers (fp8_quant.hip), products
 * (fp8_gemm.hip) and weight gradients (fp8_grad.hip) one after another on a stream. No kernel here: a call for each of them from
 * Python, with its own tensors, took 38 us forward and 31 backward of a layer whose kernels take 12 and 23 (515 x 768 x 768).
 */
#include "nanochat_amd.h"
#include "nc_fp8.h"
#include "nc_internal.h"

namespace nc {
namespace {

constexpr int NONE = -1;   /* a weight gradient that is not wanted */

bool layer_sizes(long long rows, int n, int k) {
    return rows >= 0 && n > 0 && k > 0 && n % 16 == 0 && k % 16 == 0 && n <= 1 << 20 && k <= 1 << 20 &&
           rows <= (1LL << 31) / ((k + F8_BLOCK - 1) / F8_BLOCK) - 32;
}
/* What the calls below hand on is checked before the first of them launches: a call that is refused has written nothing. */
bool bad_form(const void *codes, const void *scale, long long stride, int cols) {
    return f8_misaligned(codes, 16) || f8_bad_scales(scale, stride, cols);
}
bool bad_rows(const void *x, long long stride, long long rows, int cols) {
    return f8_misaligned(x, 2) || (rows > 1 && stride < cols) || stride > (1LL << 40);
}
long long up16(long long n) { return (n + 15) / 16 * 16; }
long long grad_need(long long rows, int n1, int n2, int mode) {
    return mode == NONE ? 0 : nc_fp8_weight_grad_workspace_bytes(rows, n1, n2);
}

}  // namespace
}  // namespace nc

using namespace nc;

extern "C" int nc_fp8_linear_fwd(const void *x, long long row_stride, const void *w, const void *w_scale, int w_scale_stride,
                                 long long rows, int n, int k, void *codes, void *scale, long long scale_stride, void *out,
                                 void *stream) {
    if (!layer_sizes(rows, n, k)) return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!x || !w || !w_scale || !codes || !scale || !out) return NC_ERR_NULL;
    if (bad_rows(x, row_stride, rows, k) || bad_form(w, w_scale, w_scale_stride, k) || bad_form(codes, scale, scale_stride, k) ||
        f8_misaligned(out, 16))
        return NC_ERR_SHAPE;
    const int status = nc_fp8_quantize_rows(x, 0, row_stride, rows, k, codes, scale, scale_stride, stream);
    return status ? status : nc_fp8_matmul(codes, scale, scale_stride, w, w_scale, w_scale_stride, rows, n, k, out, stream);
}

extern "C" long long nc_fp8_linear_bwd_workspace_bytes(long long rows, int n, int k, int need_x, int mode) {
    if (!layer_sizes(rows, n, k) || !layer_sizes(rows, k, n) || mode < NONE || mode > 2) return -1;
    const long long grad = grad_need(rows, n, k, mode);
    return grad < 0 ? -1 : (need_x ? f8_form_bytes(rows, n) : 0) + grad;
}

extern "C" int nc_fp8_linear_bwd(const void *dy, long long row_stride, const void *codes, const void *scale,
                                 long long scale_stride, const void *codes_t, const void *scale_t, int scale_t_stride,
                                 long long rows, int n, int k, void *dx, void *dw, int mode, void *workspace,
                                 long long workspace_bytes, void *stream) {
    const long long need = nc_fp8_linear_bwd_workspace_bytes(rows, n, k, dx != nullptr, mode);
    if (need < 0 || (mode != NONE && rows > 1 && row_stride != n)) return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!dy || !workspace || (dx && (!codes_t || !scale_t)) || (mode != NONE && (!codes || !scale || !dw))) return NC_ERR_NULL;
    if (bad_rows(dy, row_stride, rows, n) || (dx && (bad_form(codes_t, scale_t, scale_t_stride, n) || f8_misaligned(dx, 16))))
        return NC_ERR_SHAPE;
    if (f8_misaligned(workspace, 16) || workspace_bytes < need) return NC_ERR_WORKSPACE;
    if (mode != NONE)
        if (const int e = fp8_weight_grad_refuses({dy, codes, scale, scale_stride, n, k, mode, dw}, rows)) return e;
    int status = NC_OK;
    char *rest = (char *)workspace;
    if (dx) {
        const F8Form f(workspace, rows, n);
        rest += f.bytes;
        status = nc_fp8_quantize_rows(dy, 0, row_stride, rows, n, f.codes, f.scale, f.pitch, stream);
        if (!status)
            status = nc_fp8_matmul(f.codes, f.scale, f.pitch, codes_t, scale_t, scale_t_stride, rows, k, n, dx, stream);
    }
    if (!status && mode != NONE)
        status = nc_fp8_weight_grad(dy, codes, scale, scale_stride, rows, n, k, mode, dw, rest, need - (rest - (char *)workspace),
                                    stream);
    return status;
}

static int mlp_fwd(bool fast, const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                   const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden, int n,
                   void *codes, void *scale, long long scale_stride, void *act, void *act_scale, long long act_scale_stride,
                   void *out, void *stream) {
    if (!layer_sizes(rows, hidden, c) || !layer_sizes(rows, n, hidden)) return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    if (!x || !fc || !fc_scale || !proj || !proj_scale || !codes || !scale || !act || !act_scale || !out) return NC_ERR_NULL;
    if (bad_rows(x, row_stride, rows, c) || bad_form(fc, fc_scale, fc_scale_stride, c) ||
        bad_form(proj, proj_scale, proj_scale_stride, hidden) || bad_form(codes, scale, scale_stride, c) ||
        bad_form(act, act_scale, act_scale_stride, hidden) || f8_misaligned(out, 16))
        return NC_ERR_SHAPE;
    int status = nc_fp8_quantize_rows(x, 0, row_stride, rows, c, codes, scale, scale_stride, stream);
    if (!status)
        status = (fast ? nc_fp8_matmul_relu2_fast : nc_fp8_matmul_relu2)(codes, scale, scale_stride, fc, fc_scale, fc_scale_stride,
                                                                           rows, hidden, c, act, act_scale, act_scale_stride, stream);
    return status ? status : nc_fp8_matmul(act, act_scale, act_scale_stride, proj, proj_scale, proj_scale_stride, rows, n,
                                           hidden, out, stream);
}

extern "C" int nc_fp8_mlp_fwd(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                              const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden,
                              int n, void *codes, void *scale, long long scale_stride, void *act, void *act_scale,
                              long long act_scale_stride, void *out, void *stream) {
    return mlp_fwd(false, x, row_stride, fc, fc_scale, fc_scale_stride, proj, proj_scale, proj_scale_stride, rows, c, hidden, n, codes,
                   scale, scale_stride, act, act_scale, act_scale_stride, out, stream);
}

extern "C" int nc_fp8_mlp_fwd_fast(const void *x, long long row_stride, const void *fc, const void *fc_scale, int fc_scale_stride,
                                    const void *proj, const void *proj_scale, int proj_scale_stride, long long rows, int c, int hidden,
                                    int n, void *codes, void *scale, long long scale_stride, void *act, void *act_scale,
                                    long long act_scale_stride, void *out, void *stream) {
    return mlp_fwd(true, x, row_stride, fc, fc_scale, fc_scale_stride, proj, proj_scale, proj_scale_stride, rows, c, hidden, n, codes,
                   scale, scale_stride, act, act_scale, act_scale_stride, out, stream);
}

/* dy's form, dh, dh's form, and what the weight gradients take, one after the other. */
extern "C" long long nc_fp8_mlp_bwd_workspace_bytes(long long rows, int c, int hidden, int n, int need_x, int fc_mode,
                                                    int proj_mode) {
    if (!layer_sizes(rows, hidden, c) || !layer_sizes(rows, c, hidden) || !layer_sizes(rows, n, hidden) ||
        !layer_sizes(rows, hidden, n) || fc_mode < NONE || fc_mode > 2 || proj_mode < NONE || proj_mode > 2)
        return -1;
    const bool inner = need_x || fc_mode != NONE;
    const long long grads = fc_mode != NONE && proj_mode != NONE
                                ? fp8_weight_grads_bytes(rows, hidden, c, fc_mode, n, hidden, proj_mode)
                            : fc_mode != NONE ? grad_need(rows, hidden, c, fc_mode) : grad_need(rows, n, hidden, proj_mode);
    return grads < 0 ? -1 : (inner ? f8_form_bytes(rows, n) + up16(2 * rows * hidden) + f8_form_bytes(rows, hidden) : 0) + grads;
}

extern "C" int nc_fp8_mlp_bwd(const void *dy, long long row_stride, const void *codes, const void *scale, long long scale_stride,
                              const void *act, const void *act_scale, long long act_scale_stride, const void *fc_codes_t,
                              const void *fc_scale_t, int fc_scale_t_stride, const void *proj_codes_t, const void *proj_scale_t,
                              int proj_scale_t_stride, long long rows, int c, int hidden, int n, void *dx, void *dfc, int fc_mode,
                              void *dproj, int proj_mode, void *workspace, long long workspace_bytes, void *stream) {
    const long long need = nc_fp8_mlp_bwd_workspace_bytes(rows, c, hidden, n, dx != nullptr, fc_mode, proj_mode);
    if (need < 0 || (proj_mode != NONE && rows > 1 && row_stride != n)) return NC_ERR_SHAPE;
    if (rows == 0) return NC_OK;
    const bool inner = dx || fc_mode != NONE;
    if (!dy || !act || !act_scale || !workspace || (inner && (!proj_codes_t || !proj_scale_t)) ||
        (dx && (!fc_codes_t || !fc_scale_t)) || (fc_mode != NONE && (!codes || !scale || !dfc)) || (proj_mode != NONE && !dproj))
        return NC_ERR_NULL;
    if (bad_rows(dy, row_stride, rows, n) ||
        ((inner || proj_mode != NONE) && bad_form(act, act_scale, act_scale_stride, hidden)) ||
        (inner && bad_form(proj_codes_t, proj_scale_t, proj_scale_t_stride, n)) ||
        (dx && (bad_form(fc_codes_t, fc_scale_t, fc_scale_t_stride, hidden) || f8_misaligned(dx, 16))))
        return NC_ERR_SHAPE;
    if (f8_misaligned(workspace, 16) || workspace_bytes < need) return NC_ERR_WORKSPACE;
    GradOf g[2] = {{workspace, codes, scale, scale_stride, hidden, c, fc_mode, dfc},   /* its dy is dh, in the workspace: below */
                   {dy, act, act_scale, act_scale_stride, n, hidden, proj_mode, dproj}};
    for (const GradOf &of : g)
        if (of.mode != NONE)
            if (const int e = fp8_weight_grad_refuses(of, rows)) return e;
    int status = NC_OK;
    unsigned char *rest = (unsigned char *)workspace, *dh = nullptr;
    if (inner) {
        const F8Form f(rest, rows, n);
        dh = rest + f.bytes;
        const F8Form h(dh + up16(2 * rows * hidden), rows, hidden);
        rest = h.codes + h.bytes;
        status = nc_fp8_quantize_rows(dy, 0, row_stride, rows, n, f.codes, f.scale, f.pitch, stream);
        if (!status)
            status = nc_fp8_matmul_relu2_bwd(f.codes, f.scale, f.pitch, proj_codes_t, proj_scale_t, proj_scale_t_stride, rows,
                                             hidden, n, act, act_scale, act_scale_stride, dh, h.codes, h.scale, h.pitch, stream);
        if (!status && dx)
            status = nc_fp8_matmul(h.codes, h.scale, h.pitch, fc_codes_t, fc_scale_t, fc_scale_t_stride, rows, c, hidden, dx,
                                   stream);
    }
    const long long left = need - (rest - (unsigned char *)workspace);
    g[0].dy = dh;
    if (!status && fc_mode != NONE && proj_mode != NONE) return fp8_weight_grads(g, rows, rest, left, (hipStream_t)stream);
    if (!status && fc_mode != NONE)
        status = nc_fp8_weight_grad(dh, codes, scale, scale_stride, rows, hidden, c, fc_mode, dfc, rest, left, stream);
    if (!status && proj_mode != NONE)
        status = nc_fp8_weight_grad(dy, act, act_scale, act_scale_stride, rows, n, hidden, proj_mode, dproj, rest, left, stream);
    return status;
}
