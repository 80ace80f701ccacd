// C ABI of the MXFP4 operators and of the rows sorted by expert (declared in
// include/jjjetson_ops_amd.h).  Entries validate their arguments before they look for a
// device, launch on the caller's stream and return a status code.
#include "mxfp4_common.hpp"

using namespace jjo;

namespace {

bool aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

bool dtype_ok(int d) { return d == JJO_DTYPE_F32 || d == JJO_DTYPE_F16 || d == JJO_DTYPE_BF16; }
int elem_bytes(int d) { return d == JJO_DTYPE_F32 ? 4 : 2; }

// A launch's status; a shape whose tiles do not fit one grid is the caller's error.
int launched(hipError_t e, const char *what) {
    if (e == hipSuccess) return JJO_OK;
    if (e == hipErrorInvalidConfiguration)
        return set_error(JJO_ERR_INVALID_ARG, "%s: the shape exceeds one launch", what);
    return hip_fail(e, what);
}

int check_rows(const char *who, const void *x, int dtype, int64_t row_stride, const void *q, int64_t rows,
               int64_t cols) {
    if (x == nullptr || q == nullptr) return set_error(JJO_ERR_INVALID_ARG, "%s: null pointer argument", who);
    if (!dtype_ok(dtype)) return set_error(JJO_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    if (mxfp4_bytes(rows, cols) < 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: rows=%lld must be positive and cols=%lld a positive multiple of %d",
                         who, (long long)rows, (long long)cols, kQK);
    if (rows * (cols / 8) > kMxMaxGroups)
        return set_error(JJO_ERR_INVALID_ARG, "%s: %lld x %lld exceeds one launch", who, (long long)rows, (long long)cols);
    if (!aligned(x, 16) || !aligned(q, 16))
        return set_error(JJO_ERR_INVALID_ARG, "%s: 16-byte aligned buffers required", who);
    if (rows > 1 && (row_stride < cols || row_stride > (1LL << 40) || row_stride * elem_bytes(dtype) % 16 != 0))
        return set_error(JJO_ERR_INVALID_ARG,
                         "%s: row_stride=%lld must be at least cols=%lld and keep rows 16-byte aligned", who,
                         (long long)row_stride, (long long)cols);
    return JJO_OK;
}

int check_mm(const char *who, const void *w, const void *x, const void *y, int dtype, int K, int N, int M) {
    if (w == nullptr || x == nullptr || y == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "%s: null pointer argument", who);
    if (!dtype_ok(dtype)) return set_error(JJO_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    if (K <= 0 || N <= 0 || M <= 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: ncols_k=%d nrows_out=%d batch=%d must be positive", who, K, N, M);
    if (K % kQK != 0) return set_error(JJO_ERR_INVALID_ARG, "%s: ncols_k=%d must be a multiple of %d", who, K, kQK);
    if (M > 1 << 28 || N > 1 << 28 || K > 1 << 28)
        return set_error(JJO_ERR_INVALID_ARG, "%s: ncols_k=%d nrows_out=%d batch=%d: at most 2^28 each", who, K, N, M);
    if (!aligned(w, 16) || !aligned(x, 16) || !aligned(y, 16))
        return set_error(JJO_ERR_INVALID_ARG, "%s: 16-byte aligned buffers required", who);
    return JJO_OK;
}

int check_experts(const char *who, const void *offsets, int n_experts) {
    if (offsets == nullptr || n_experts <= 0 || n_experts > 4096)
        return set_error(JJO_ERR_INVALID_ARG, "%s: expert_offsets and 1 <= num_experts <= 4096 required (got %d)", who,
                         n_experts);
    return JJO_OK;
}

int check_routes(const char *who, int dtype, int T, int H, int E, int top_k) {
    if (!dtype_ok(dtype)) return set_error(JJO_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    if (T <= 0 || H <= 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: num_tokens=%d hidden_size=%d must be positive", who, T, H);
    if (E <= 0 || E > 1024 || top_k <= 0 || top_k > 32)
        return set_error(JJO_ERR_INVALID_ARG, "%s: need 1 <= top_k <= 32 and 1 <= num_experts <= 1024 (got top_k=%d "
                         "num_experts=%d)", who, top_k, E);
    if (T > (1 << 23) || (int64_t)T * top_k > 1 << 26 || H > 1 << 23)
        return set_error(JJO_ERR_INVALID_ARG, "%s: num_tokens=%d, top_k=%d, hidden_size=%d exceed one launch", who, T,
                         top_k, H);
    return JJO_OK;
}

struct MxFfnWs {
    float *route_w;
    int32_t *ids, *offsets, *src_route, *dst_of_route;
    uint8_t *xq, *midq;
    float *eout;
    int slices;  // of the down product, each R rows of eout
    int64_t bytes;
};

MxFfnWs ffn_layout(uint8_t *base, int T, int H, int I, int E, int top_k) {
    const int64_t R = (int64_t)T * top_k;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        uint8_t *p = base ? base + off : nullptr;
        off += (bytes + 255) / 256 * 256;
        return p;
    };
    MxFfnWs w{};
    w.route_w = (float *)take(R * 4);
    w.ids = (int32_t *)take(R * 4);
    w.offsets = (int32_t *)take((int64_t)(E + 1) * 4);
    w.src_route = (int32_t *)take(R * 4);
    w.dst_of_route = (int32_t *)take(R * 4);
    w.xq = take(mx_bytes(T, H));
    w.midq = take(mx_bytes(R, I));
    w.slices = mxfp4_down_slices(I, H, (int)R, E);
    w.eout = (float *)take(w.slices * R * H * 4);
    w.bytes = off;
    return w;
}

int check_ffn(int T, int H, int I, int E, int top_k) {
    const int rc = check_routes("moe_mxfp4_ffn", JJO_DTYPE_F32, T, H, E, top_k);
    if (rc != JJO_OK) return rc;
    if (H % kQK != 0 || I <= 0 || I % kQK != 0 || I > 1 << 28 || top_k > E)
        return set_error(JJO_ERR_INVALID_ARG, "moe_mxfp4_ffn: hidden_size=%d and intermediate_size=%d must be positive "
                         "multiples of %d, top_k=%d at most num_experts=%d", H, I, kQK, top_k, E);
    return JJO_OK;
}

}  // namespace

extern "C" {

int64_t mxfp4_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols % kQK != 0 || rows > (1LL << 56) / cols) return -1;
    return mx_bytes(rows, cols);
}

int quantize_mxfp4_device(void *stream, const void *x, int dtype, int64_t row_stride, void *out, int64_t rows,
                          int64_t cols) {
    clear_error();
    int rc = check_rows("quantize_mxfp4", x, dtype, row_stride, out, rows, cols);
    if (rc != JJO_OK || (rc = require_device()) != JJO_OK) return rc;
    return launched(launch_quantize_mxfp4(x, dtype, row_stride, out, rows, cols, (hipStream_t)stream),
                    "quantize_mxfp4 launch");
}

int dequantize_mxfp4_device(void *stream, const void *q, void *y, int dtype, int64_t row_stride, int64_t rows,
                            int64_t cols) {
    clear_error();
    int rc = check_rows("dequantize_mxfp4", y, dtype, row_stride, q, rows, cols);
    if (rc != JJO_OK || (rc = require_device()) != JJO_OK) return rc;
    return launched(launch_dequantize_mxfp4(q, y, dtype, row_stride, rows, cols, (hipStream_t)stream),
                    "dequantize_mxfp4 launch");
}

int mat_mul_mxfp4_device(const void *d_w, const void *d_x_mxfp4, void *d_y, int y_dtype, int ncols_k, int nrows_out,
                         int batch, void *stream) {
    clear_error();
    int rc = check_mm("mat_mul_mxfp4", d_w, d_x_mxfp4, d_y, y_dtype, ncols_k, nrows_out, batch);
    if (rc != JJO_OK || (rc = require_device()) != JJO_OK) return rc;
    return launched(launch_mxfp4_mm(d_w, d_x_mxfp4, d_y, y_dtype, ncols_k, nrows_out, batch, MxGroups{},
                                        (hipStream_t)stream),
                    "mat_mul_mxfp4 launch");
}

int64_t linear_mxfp4_workspace_bytes(int in_features, int num_tokens) {
    const int64_t bytes = mxfp4_bytes(num_tokens, in_features);
    return bytes >= 0 && num_tokens == 1 && in_features <= kMxFusedMaxK ? 0 : bytes;
}

int linear_mxfp4_forward_device(void *stream, void *quant_workspace, const void *input, int in_dtype,
                                const void *weight, void *output, int out_dtype, int in_features, int out_features,
                                int num_tokens) {
    clear_error();
    int rc = check_mm("linear_mxfp4", weight, input, output, out_dtype, in_features, out_features, num_tokens);
    if (rc != JJO_OK) return rc;
    if (!dtype_ok(in_dtype)) return set_error(JJO_ERR_INVALID_ARG, "linear_mxfp4: unknown dtype %d", in_dtype);
    const bool fused = num_tokens == 1 && in_features <= kMxFusedMaxK;
    if (!fused && (quant_workspace == nullptr || !aligned(quant_workspace, 16)))
        return set_error(JJO_ERR_INVALID_ARG, "linear_mxfp4: a 16-byte aligned workspace is required");
    if ((rc = require_device()) != JJO_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (fused)
        return launched(launch_mxfp4_gemv(weight, input, in_dtype, output, out_dtype, in_features, out_features, s),
                        "linear_mxfp4 launch");
    const hipError_t e = launch_quantize_mxfp4(input, in_dtype, in_features, quant_workspace, num_tokens, in_features, s);
    if (e != hipSuccess) return launched(e, "linear_mxfp4 quantize");
    return launched(launch_mxfp4_mm(weight, quant_workspace, output, out_dtype, in_features, out_features,
                                        num_tokens, MxGroups{}, s),
                    "linear_mxfp4 launch");
}

int mat_mul_mxfp4_grouped_device(const void *d_w, const void *d_x_mxfp4, const int32_t *d_expert_offsets,
                                 int n_experts, const int32_t *d_route_dst, void *d_y, int y_dtype, int ncols_k,
                                 int nrows_out, int n_routes, void *stream) {
    clear_error();
    int rc = check_mm("mat_mul_mxfp4_grouped", d_w, d_x_mxfp4, d_y, y_dtype, ncols_k, nrows_out, n_routes);
    if (rc != JJO_OK || (rc = check_experts("mat_mul_mxfp4_grouped", d_expert_offsets, n_experts)) != JJO_OK ||
        (rc = require_device()) != JJO_OK)
        return rc;
    MxGroups g;
    g.offsets = d_expert_offsets, g.n_experts = n_experts, g.route_dst = d_route_dst;
    return launched(launch_mxfp4_mm(d_w, d_x_mxfp4, d_y, y_dtype, ncols_k, nrows_out, n_routes, g,
                                        (hipStream_t)stream),
                    "mat_mul_mxfp4_grouped launch");
}

int moe_mxfp4_gate_up_swiglu_device(void *stream, const void *w_gate, const void *w_up, const void *x_mxfp4_permuted,
                                    const int32_t *expert_offsets, int num_experts, void *mid_mxfp4, int hidden_size,
                                    int intermediate_size, int n_routes) {
    clear_error();
    const char *who = "moe_mxfp4_gate_up_swiglu";
    int rc = check_mm(who, w_gate, x_mxfp4_permuted, mid_mxfp4, JJO_DTYPE_F32, hidden_size, intermediate_size, n_routes);
    if (rc != JJO_OK || (rc = check_experts(who, expert_offsets, num_experts)) != JJO_OK) return rc;
    if (w_up == nullptr || !aligned(w_up, 16) || intermediate_size % kQK != 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: a 16-byte aligned w_up and intermediate_size=%d a multiple of %d "
                         "required", who, intermediate_size, kQK);
    if ((rc = require_device()) != JJO_OK) return rc;
    MxGroups g;
    g.offsets = expert_offsets, g.n_experts = num_experts;
    return launched(launch_mxfp4_swiglu(w_gate, w_up, x_mxfp4_permuted, mid_mxfp4, hidden_size,
                                               intermediate_size, n_routes, g, (hipStream_t)stream),
                    who);
}

int64_t moe_mxfp4_ffn_workspace_bytes(int num_tokens, int hidden_size, int intermediate_size, int num_experts,
                                      int top_k) {
    clear_error();
    if (check_ffn(num_tokens, hidden_size, intermediate_size, num_experts, top_k) != JJO_OK) return -1;
    return ffn_layout(nullptr, num_tokens, hidden_size, intermediate_size, num_experts, top_k).bytes;
}

int moe_mxfp4_ffn_forward_device(void *stream, const void *x, const float *logits, const void *w_gate,
                                 const void *w_up, const void *w_down, void *y, int dtype, int num_tokens,
                                 int hidden_size, int intermediate_size, int num_experts, int top_k, void *workspace,
                                 int64_t workspace_bytes) {
    clear_error();
    const int T = num_tokens, H = hidden_size, I = intermediate_size, E = num_experts;
    int rc = check_ffn(T, H, I, E, top_k);
    if (rc != JJO_OK) return rc;
    const int R = T * top_k;
    if (!dtype_ok(dtype)) return set_error(JJO_ERR_INVALID_ARG, "moe_mxfp4_ffn: unknown dtype %d", dtype);
    for (const void *p : {x, (const void *)logits, w_gate, w_up, w_down, (const void *)y, (const void *)workspace})
        if (p == nullptr) return set_error(JJO_ERR_INVALID_ARG, "moe_mxfp4_ffn: null pointer argument");
    if (!aligned(x, 16) || !aligned(y, 16) || !aligned(w_gate, 16) || !aligned(w_up, 16) || !aligned(w_down, 16) ||
        !aligned(logits, 4) || !aligned(workspace, 256))
        return set_error(JJO_ERR_INVALID_ARG, "moe_mxfp4_ffn: x, y and weights 16-byte, workspace 256-byte aligned");
    const MxFfnWs ws = ffn_layout((uint8_t *)workspace, T, H, I, E, top_k);
    if (workspace_bytes < ws.bytes)
        return set_error(JJO_ERR_INVALID_ARG, "moe_mxfp4_ffn: workspace of %lld bytes, need %lld",
                         (long long)workspace_bytes, (long long)ws.bytes);
    if ((rc = require_device()) != JJO_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    // 1) top-k, sort, and x to MXFP4 once per token (the products fetch a route's row by its token),
    // 2) gate|up with SwiGLU, 3) down, 4) weighted sum back to token order
    MxGroups g;
    g.offsets = ws.offsets, g.n_experts = E;
    hipError_t e = launch_mxfp4_route(x, dtype, logits, T, H, E, top_k, ws.route_w, ws.ids, ws.offsets, ws.src_route,
                                      ws.dst_of_route, ws.xq, s);
    if (e != hipSuccess) return launched(e, "moe_mxfp4_ffn routing");
    g.src_route = ws.src_route, g.top_k = top_k, g.x_rows = T;
    if ((e = launch_mxfp4_swiglu(w_gate, w_up, ws.xq, ws.midq, H, I, R, g, s)) != hipSuccess)
        return launched(e, "moe_mxfp4_ffn gate|up");
    g.src_route = nullptr;
    if ((e = launch_mxfp4_mm(w_down, ws.midq, ws.eout, JJO_DTYPE_F32, I, H, R, g, s, ws.slices)) != hipSuccess)
        return launched(e, "moe_mxfp4_ffn down");
    return launched(launch_moe_join_rows(ws.eout, JJO_DTYPE_F32, ws.dst_of_route, ws.route_w, y, dtype, T, H, top_k, s,
                                         ws.slices),
                    "moe_mxfp4_ffn combine");
}

int moe_dispatch_rows_device(void *stream, const int32_t *expert_ids, const void *x, int dtype, int num_tokens,
                             int top_k, int hidden_size, int num_experts, int32_t *expert_offsets,
                             int32_t *src_route, int32_t *dst_of_route, void *x_sorted) {
    clear_error();
    int rc = check_routes("moe_dispatch_rows", dtype, num_tokens, hidden_size, num_experts, top_k);
    if (rc != JJO_OK) return rc;
    if (expert_ids == nullptr || x == nullptr || expert_offsets == nullptr || src_route == nullptr ||
        dst_of_route == nullptr || x_sorted == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "moe_dispatch_rows: null pointer argument");
    if ((rc = require_device()) != JJO_OK) return rc;
    return launched(launch_moe_dispatch_rows(expert_ids, x, elem_bytes(dtype), num_tokens, top_k, hidden_size,
                                             num_experts, expert_offsets, src_route, dst_of_route, x_sorted,
                                             (hipStream_t)stream),
                    "moe_dispatch_rows launch");
}

int moe_dispatch_rows_backward_device(void *stream, const void *grad_sorted, int dtype, const int32_t *dst_of_route,
                                      void *grad_x, int num_tokens, int hidden_size, int top_k) {
    clear_error();
    int rc = check_routes("moe_dispatch_rows_backward", dtype, num_tokens, hidden_size, 1, top_k);
    if (rc != JJO_OK) return rc;
    if (grad_sorted == nullptr || dst_of_route == nullptr || grad_x == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "moe_dispatch_rows_backward: null pointer argument");
    if ((rc = require_device()) != JJO_OK) return rc;
    return launched(launch_moe_join_rows(grad_sorted, dtype, dst_of_route, nullptr, grad_x, dtype, num_tokens,
                                         hidden_size, top_k, (hipStream_t)stream),
                    "moe_dispatch_rows_backward launch");
}

int moe_combine_rows_device(void *stream, const void *expert_out, int dtype, const int32_t *dst_of_route,
                            const float *route_weights, void *y, int num_tokens, int hidden_size, int top_k) {
    clear_error();
    int rc = check_routes("moe_combine_rows", dtype, num_tokens, hidden_size, 1, top_k);
    if (rc != JJO_OK) return rc;
    if (expert_out == nullptr || dst_of_route == nullptr || route_weights == nullptr || y == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "moe_combine_rows: null pointer argument");
    if ((rc = require_device()) != JJO_OK) return rc;
    return launched(launch_moe_join_rows(expert_out, dtype, dst_of_route, route_weights, y, dtype, num_tokens,
                                         hidden_size, top_k, (hipStream_t)stream),
                    "moe_combine_rows launch");
}

int moe_combine_rows_backward_device(void *stream, const void *grad_y, const void *expert_out, int dtype,
                                     const int32_t *dst_of_route, const float *route_weights, void *grad_expert_out,
                                     float *grad_route_weights, int num_tokens, int hidden_size, int top_k) {
    clear_error();
    int rc = check_routes("moe_combine_rows_backward", dtype, num_tokens, hidden_size, 1, top_k);
    if (rc != JJO_OK) return rc;
    for (const void *p : {grad_y, expert_out, (const void *)dst_of_route, (const void *)route_weights,
                          (const void *)grad_expert_out, (const void *)grad_route_weights})
        if (p == nullptr) return set_error(JJO_ERR_INVALID_ARG, "moe_combine_rows_backward: null pointer argument");
    if ((rc = require_device()) != JJO_OK) return rc;
    return launched(launch_moe_combine_rows_backward(grad_y, expert_out, dtype, dst_of_route, route_weights,
                                                     grad_expert_out, grad_route_weights, num_tokens, hidden_size,
                                                     top_k, (hipStream_t)stream),
                    "moe_combine_rows_backward launch");
}

}  // extern "C"
