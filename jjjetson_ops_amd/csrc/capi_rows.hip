// C ABI of the products of float matrices (declared in include/jjjetson_ops_amd.h): a linear layer with
// bias, activation and residual, the experts' products of sorted rows, gate|up with SwiGLU, and their
// gradients.  Entries validate their arguments before they look for a device, launch on the caller's
// stream and return a status code.
#include "rows_mm.hpp"

using namespace jjo;

namespace {

constexpr int64_t kMaxStride = 1LL << 40;

bool dtype_ok(int d) { return d == JJO_DTYPE_F32 || d == JJO_DTYPE_F16 || d == JJO_DTYPE_BF16; }
int elem_bytes(int d) { return d == JJO_DTYPE_F32 ? 4 : 2; }
int64_t up256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int launched(hipError_t e, const char *what) {
    if (e == hipSuccess) return JJO_OK;
    if (e == hipErrorInvalidConfiguration)
        return set_error(JJO_ERR_INVALID_ARG, "%s: the shape exceeds one launch", what);
    return hip_fail(e, what);
}

// K, N and rows of a product; at most 2^28 each and 2^40 elements of any of its matrices.
int check_sizes(const char *who, int dtype, int K, int N, int rows, int n_experts) {
    if (!dtype_ok(dtype)) return set_error(JJO_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    if (K <= 0 || N <= 0 || rows <= 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: sizes %d, %d and %d rows must be positive", who, K, N, rows);
    if (K > 1 << 28 || N > 1 << 28 || rows > 1 << 28)
        return set_error(JJO_ERR_INVALID_ARG, "%s: sizes %d, %d and %d rows: at most 2^28 each", who, K, N, rows);
    if (n_experts <= 0 || n_experts > 4096)
        return set_error(JJO_ERR_INVALID_ARG, "%s: 1 <= num_experts <= 4096 required (got %d)", who, n_experts);
    if ((int64_t)K * N > kMaxStride / n_experts || (int64_t)K * rows > kMaxStride || (int64_t)N * rows > kMaxStride)
        return set_error(JJO_ERR_INVALID_ARG, "%s: a matrix of more than 2^40 elements", who);
    return JJO_OK;
}

// A pointer that may not be null, or may be, aligned to its elements.
int check_ptr(const char *who, const char *name, const void *p, int align, bool may_be_null = false) {
    if (p == nullptr)
        return may_be_null ? JJO_OK : set_error(JJO_ERR_INVALID_ARG, "%s: %s is a null pointer", who, name);
    if ((uintptr_t)p % (unsigned)align != 0)
        return set_error(JJO_ERR_INVALID_ARG, "%s: %s must be aligned to its elements (%d bytes)", who, name, align);
    return JJO_OK;
}

int check_stride(const char *who, const char *name, int64_t stride, int cols, int rows) {
    if (rows > 1 && (stride < cols || stride > kMaxStride / rows))
        return set_error(JJO_ERR_INVALID_ARG, "%s: %s=%lld must be at least %d, %d rows within 2^40 elements", who,
                         name, (long long)stride, cols, rows);
    return JJO_OK;
}

int check_workspace(const char *who, const void *ws, int64_t have, int64_t need) {
    if (need == 0) return JJO_OK;
    if (ws == nullptr || have < need)
        return set_error(JJO_ERR_INVALID_ARG, "%s: workspace of %lld bytes, need %lld", who,
                         ws == nullptr ? 0LL : (long long)have, (long long)need);
    if ((uintptr_t)ws % 256 != 0) return set_error(JJO_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", who);
    return JJO_OK;
}

int check_activation(const char *who, int activation) {
    if (activation < JJO_ACT_NONE || activation > JJO_ACT_SILU)
        return set_error(JJO_ERR_INVALID_ARG, "%s: unknown activation %d", who, activation);
    return JJO_OK;
}

int check_grad_dtype(const char *who, int grad_dtype, int dtype) {
    if (grad_dtype != dtype && grad_dtype != JJO_DTYPE_F32)
        return set_error(JJO_ERR_INVALID_ARG, "%s: gradients of the weights are of the weights' dtype or fp32", who);
    return JJO_OK;
}

#define JJO_TRY(call)                         \
    do {                                      \
        const int jjo_rc_ = (call);           \
        if (jjo_rc_ != JJO_OK) return jjo_rc_; \
    } while (0)

// A row's stride where there is one row only: any value is accepted, none is used.
int64_t stride_of(int64_t stride, int cols, int rows) { return rows > 1 ? stride : cols; }

// ---- the products, without pointers to the operands
RowsMm product(RowsMode mode, int dtype, int P, int Q, int K, int halves, int n_experts) {
    RowsMm m{};
    m.P = P, m.Q = Q, m.K = K, m.halves = halves, m.terms = 1;
    m.n_experts = n_experts;
    m.M = mode == kRowsWeight ? K : Q;
    m.slices = rows_mm_choose(mode, dtype, P, Q, K, halves, n_experts).slices;
    return m;
}

// n_experts 0: one matrix.  Forward [rows][K] -> [rows][N].
RowsMm forward(int dtype, int K, int N, int rows, int n_experts) {
    RowsMm m = product(kRowsForward, dtype, N, rows, K, 1, n_experts);
    m.ldp = K, m.ldq = K, m.ldy = N, m.expert_stride = (int64_t)N * K;
    return m;
}
RowsMm swiglu(int dtype, int H, int I, int rows, int n_experts) {
    RowsMm m = product(kRowsSwiglu, dtype, I, rows, H, 1, n_experts);
    m.ldp = H, m.ldq = H, m.ldy = I, m.expert_stride = (int64_t)I * H;
    return m;
}
// [rows][halves * N] -> [rows][K]
RowsMm input(int dtype, int K, int N, int rows, int n_experts, int halves) {
    RowsMm m = product(kRowsInput, dtype, K, rows, N, halves, n_experts);
    m.ldp = K, m.ldq = (int64_t)halves * N, m.ldy = K, m.expert_stride = (int64_t)N * K;
    return m;
}
// [rows][halves * N], [rows][K] -> halves x [N][K]
RowsMm weight(int dtype, int K, int N, int rows, int n_experts, int halves, bool wide) {
    RowsMm m = product(kRowsWeight, dtype, K, N, rows, halves, n_experts);
    m.ldp = K, m.ldq = (int64_t)halves * N, m.ldy = K, m.expert_stride = (int64_t)N * K, m.wide = wide;
    return m;
}

// The gradient through an activation, rounded to `dtype`.  Where the weights' gradients are fp32 and it is not, what
// the rounding left is kept as well, rounded again: two terms of fp16 are 22 bits (below 2^-14, fp16's smallest
// normal number, the second ends at 2^-36, and the matrix unit's additions are as exact as those of 2^-14), three of
// bf16 24.
int64_t gz_plane_bytes(int dtype, int64_t values) { return up256(elem_bytes(dtype) * values); }
int gz_planes(int dtype) { return dtype == JJO_DTYPE_F32 ? 1 : dtype == JJO_DTYPE_F16 ? 2 : 3; }

// The terms of a weight's gradient, planes of gz, the smallest first.
void terms_of_gz(RowsMm &m, const uint8_t *gz, int64_t plane, int planes, int es) {
    m.terms = planes;
    m.q = gz + (planes - 1) * plane;
    if (planes > 1) m.rest = gz + (planes - 2) * plane, m.rest_plane = -plane / es;
    if (planes == 2) m.first_scale = 1.0f / kRowsRestScale;
}

// What a backward pass is asked for, and with it what its workspace holds.
struct Wanted {
    bool rows, weights, bias;
};
constexpr Wanted kAll{true, true, true};

// Sums in slices of the products asked for, one after the other in the same place (n_experts 0: one matrix).
int64_t part_bytes(int dtype, int K, int N, int rows, int n_experts, int halves, Wanted want) {
    const int64_t a = want.rows ? rows_part_bytes(kRowsInput, input(dtype, K, N, rows, n_experts, halves)) : 0;
    const int64_t b =
        want.weights ? rows_part_bytes(kRowsWeight, weight(dtype, K, N, rows, n_experts, halves, false)) : 0;
    return up256(std::max(a, b));
}

// Planes of gz: none without an activation.
int planes_of(int dtype, int grad_weight_dtype, bool act, bool weights) {
    return !act ? 0 : weights && grad_weight_dtype != dtype ? gz_planes(dtype) : 1;
}

struct LinearBackwardWs {
    int64_t gz, plane, columns, parts, bytes;  // offsets; bytes of a plane of gz
};
LinearBackwardWs linear_backward_ws(int dtype, int K, int N, int T, int planes, Wanted want) {
    LinearBackwardWs w{};
    w.plane = gz_plane_bytes(dtype, (int64_t)T * N);
    w.columns = planes * w.plane;
    w.parts = w.columns + (want.bias ? up256(4LL * rows_column_chunks(T, N) * N) : 0);
    w.bytes = w.parts + part_bytes(dtype, K, N, T, 0, 1, want);
    return w;
}
int64_t swiglu_backward_bytes(int dtype, int H, int I, int rows, int n_experts, int planes, Wanted want) {
    return planes * gz_plane_bytes(dtype, 2LL * rows * I) + part_bytes(dtype, H, I, rows, n_experts, 2, want);
}

}  // namespace

extern "C" {

int64_t linear_rows_workspace_bytes(int dtype, int in_features, int out_features, int num_tokens) {
    clear_error();
    if (check_sizes("linear_rows", dtype, in_features, out_features, num_tokens, 1) != JJO_OK) return -1;
    return rows_part_bytes(kRowsForward, forward(dtype, in_features, out_features, num_tokens, 0));
}

int linear_rows_forward_device(void *stream, const void *x, int64_t x_stride, const void *weight_, const void *bias,
                               const void *residual, int64_t residual_stride, void *y, int64_t y_stride, void *pre,
                               int dtype, int activation, int in_features, int out_features, int num_tokens,
                               void *workspace, int64_t workspace_bytes) {
    clear_error();
    const char *who = "linear_rows";
    const int K = in_features, N = out_features, T = num_tokens;
    JJO_TRY(check_sizes(who, dtype, K, N, T, 1));
    const int es = elem_bytes(dtype);
    JJO_TRY(check_activation(who, activation));
    JJO_TRY(check_ptr(who, "x", x, es));
    JJO_TRY(check_ptr(who, "weight", weight_, es));
    JJO_TRY(check_ptr(who, "bias", bias, es, true));
    JJO_TRY(check_ptr(who, "residual", residual, es, true));
    JJO_TRY(check_ptr(who, "y", y, es));
    JJO_TRY(check_ptr(who, "pre", pre, es, true));
    JJO_TRY(check_stride(who, "x_stride", x_stride, K, T));
    if (residual != nullptr) JJO_TRY(check_stride(who, "residual_stride", residual_stride, N, T));
    JJO_TRY(check_stride(who, "y_stride", y_stride, N, T));
    RowsMm m = forward(dtype, K, N, T, 0);
    JJO_TRY(check_workspace(who, workspace, workspace_bytes, rows_part_bytes(kRowsForward, m)));
    JJO_TRY(require_device());
    m.p = weight_, m.q = x, m.ldq = stride_of(x_stride, K, T);
    m.y = y, m.ldy = stride_of(y_stride, N, T);
    m.epi.bias = bias, m.epi.residual = residual, m.epi.residual_stride = stride_of(residual_stride, N, T);
    m.epi.pre = pre, m.epi.act = activation;
    m.part = (float *)workspace;
    return launched(launch_rows_mm(kRowsForward, dtype, m, (hipStream_t)stream), "linear_rows launch");
}

int64_t linear_rows_backward_workspace_bytes(int dtype, int in_features, int out_features, int num_tokens) {
    clear_error();
    if (check_sizes("linear_rows_backward", dtype, in_features, out_features, num_tokens, 1) != JJO_OK) return -1;
    return linear_backward_ws(dtype, in_features, out_features, num_tokens, gz_planes(dtype), kAll).bytes;
}

int64_t linear_rows_backward_workspace_bytes_for(int dtype, int grad_weight_dtype, int activation, int in_features,
                                                 int out_features, int num_tokens) {
    clear_error();
    const char *who = "linear_rows_backward";
    if (check_sizes(who, dtype, in_features, out_features, num_tokens, 1) != JJO_OK ||
        check_grad_dtype(who, grad_weight_dtype, dtype) != JJO_OK || check_activation(who, activation) != JJO_OK)
        return -1;
    const int planes = planes_of(dtype, grad_weight_dtype, activation != JJO_ACT_NONE, true);
    return linear_backward_ws(dtype, in_features, out_features, num_tokens, planes, kAll).bytes;
}

int linear_rows_backward_device(void *stream, const void *grad_y, int64_t grad_y_stride, const void *x,
                                int64_t x_stride, const void *weight_, const void *pre, void *grad_x,
                                int64_t grad_x_stride, void *grad_weight, void *grad_bias, int dtype,
                                int grad_weight_dtype, int activation, int in_features, int out_features,
                                int num_tokens, void *workspace, int64_t workspace_bytes) {
    clear_error();
    const char *who = "linear_rows_backward";
    const int K = in_features, N = out_features, T = num_tokens;
    JJO_TRY(check_sizes(who, dtype, K, N, T, 1));
    JJO_TRY(check_grad_dtype(who, grad_weight_dtype, dtype));
    const int es = elem_bytes(dtype), ges = elem_bytes(grad_weight_dtype);
    const bool wide = grad_weight_dtype == JJO_DTYPE_F32, act = activation != JJO_ACT_NONE;
    JJO_TRY(check_activation(who, activation));
    if (grad_x == nullptr && grad_weight == nullptr && grad_bias == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "%s: no gradient is asked for", who);
    JJO_TRY(check_ptr(who, "grad_y", grad_y, es));
    JJO_TRY(check_ptr(who, "x", x, es, grad_weight == nullptr));
    JJO_TRY(check_ptr(who, "weight", weight_, es, grad_x == nullptr));
    JJO_TRY(check_ptr(who, "pre", pre, es, !act));
    JJO_TRY(check_ptr(who, "grad_x", grad_x, es, true));
    JJO_TRY(check_ptr(who, "grad_weight", grad_weight, ges, true));
    JJO_TRY(check_ptr(who, "grad_bias", grad_bias, ges, true));
    JJO_TRY(check_stride(who, "grad_y_stride", grad_y_stride, N, T));
    if (grad_weight != nullptr) JJO_TRY(check_stride(who, "x_stride", x_stride, K, T));
    if (grad_x != nullptr) JJO_TRY(check_stride(who, "grad_x_stride", grad_x_stride, K, T));
    const int planes = planes_of(dtype, grad_weight_dtype, act, grad_weight != nullptr);
    const LinearBackwardWs ws =
        linear_backward_ws(dtype, K, N, T, planes, {grad_x != nullptr, grad_weight != nullptr, grad_bias != nullptr});
    JJO_TRY(check_workspace(who, workspace, workspace_bytes, ws.bytes));
    JJO_TRY(require_device());
    hipStream_t s = (hipStream_t)stream;
    uint8_t *const base = (uint8_t *)workspace;
    const void *gz = grad_y;
    int64_t gz_stride = stride_of(grad_y_stride, N, T);
    if (act || grad_bias != nullptr) {
        const hipError_t e =
            launch_rows_act_backward(grad_y, gz_stride, pre, base + ws.gz, planes, ws.plane / es, dtype, activation,
                                     grad_bias, wide, (float *)(base + ws.columns), T, N, s);
        if (e != hipSuccess) return launched(e, "linear_rows_backward activation");
        if (act) gz = base + ws.gz, gz_stride = N;
    }
    if (grad_x != nullptr) {
        RowsMm m = input(dtype, K, N, T, 0, 1);
        m.p = weight_, m.q = gz, m.ldq = gz_stride, m.y = grad_x, m.ldy = stride_of(grad_x_stride, K, T);
        m.part = (float *)(base + ws.parts);
        const hipError_t e = launch_rows_mm(kRowsInput, dtype, m, s);
        if (e != hipSuccess) return launched(e, "linear_rows_backward input");
    }
    if (grad_weight != nullptr) {
        RowsMm m = weight(dtype, K, N, T, 0, 1, wide);
        m.p = x, m.ldp = stride_of(x_stride, K, T), m.q = gz, m.ldq = gz_stride, m.y = grad_weight;
        if (act) terms_of_gz(m, base + ws.gz, ws.plane, planes, es);
        m.part = (float *)(base + ws.parts);
        const hipError_t e = launch_rows_mm(kRowsWeight, dtype, m, s);
        if (e != hipSuccess) return launched(e, "linear_rows_backward weight");
    }
    return JJO_OK;
}

int64_t mat_mul_rows_grouped_workspace_bytes(int dtype, int ncols_k, int nrows_out, int n_routes, int n_experts) {
    clear_error();
    if (check_sizes("mat_mul_rows_grouped", dtype, ncols_k, nrows_out, n_routes, n_experts) != JJO_OK) return -1;
    return rows_part_bytes(kRowsForward, forward(dtype, ncols_k, nrows_out, n_routes, n_experts));
}

int mat_mul_rows_grouped_device(void *stream, const void *x_sorted, const void *weights, const int32_t *expert_offsets,
                                int n_experts, void *y, int dtype, int ncols_k, int nrows_out, int n_routes,
                                void *workspace, int64_t workspace_bytes) {
    clear_error();
    const char *who = "mat_mul_rows_grouped";
    JJO_TRY(check_sizes(who, dtype, ncols_k, nrows_out, n_routes, n_experts));
    const int es = elem_bytes(dtype);
    JJO_TRY(check_ptr(who, "x_sorted", x_sorted, es));
    JJO_TRY(check_ptr(who, "weights", weights, es));
    JJO_TRY(check_ptr(who, "expert_offsets", expert_offsets, 4));
    JJO_TRY(check_ptr(who, "y", y, es));
    RowsMm m = forward(dtype, ncols_k, nrows_out, n_routes, n_experts);
    JJO_TRY(check_workspace(who, workspace, workspace_bytes, rows_part_bytes(kRowsForward, m)));
    JJO_TRY(require_device());
    m.p = weights, m.q = x_sorted, m.y = y, m.offsets = expert_offsets, m.part = (float *)workspace;
    return launched(launch_rows_mm(kRowsForward, dtype, m, (hipStream_t)stream), "mat_mul_rows_grouped launch");
}

int64_t mat_mul_rows_grouped_backward_workspace_bytes(int dtype, int ncols_k, int nrows_out, int n_routes,
                                                      int n_experts) {
    clear_error();
    if (check_sizes("mat_mul_rows_grouped_backward", dtype, ncols_k, nrows_out, n_routes, n_experts) != JJO_OK)
        return -1;
    return part_bytes(dtype, ncols_k, nrows_out, n_routes, n_experts, 1, kAll);
}

int mat_mul_rows_grouped_backward_device(void *stream, const void *grad_y, const void *x_sorted, const void *weights,
                                         const int32_t *expert_offsets, int n_experts, void *grad_x_sorted,
                                         void *grad_weights, int dtype, int grad_weights_dtype, int ncols_k,
                                         int nrows_out, int n_routes, void *workspace, int64_t workspace_bytes) {
    clear_error();
    const char *who = "mat_mul_rows_grouped_backward";
    JJO_TRY(check_sizes(who, dtype, ncols_k, nrows_out, n_routes, n_experts));
    JJO_TRY(check_grad_dtype(who, grad_weights_dtype, dtype));
    const int es = elem_bytes(dtype);
    if (grad_x_sorted == nullptr && grad_weights == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "%s: no gradient is asked for", who);
    JJO_TRY(check_ptr(who, "grad_y", grad_y, es));
    JJO_TRY(check_ptr(who, "x_sorted", x_sorted, es, grad_weights == nullptr));
    JJO_TRY(check_ptr(who, "weights", weights, es, grad_x_sorted == nullptr));
    JJO_TRY(check_ptr(who, "expert_offsets", expert_offsets, 4));
    JJO_TRY(check_ptr(who, "grad_x_sorted", grad_x_sorted, es, true));
    JJO_TRY(check_ptr(who, "grad_weights", grad_weights, elem_bytes(grad_weights_dtype), true));
    JJO_TRY(check_workspace(who, workspace, workspace_bytes,
                            part_bytes(dtype, ncols_k, nrows_out, n_routes, n_experts, 1,
                                       {grad_x_sorted != nullptr, grad_weights != nullptr, false})));
    JJO_TRY(require_device());
    hipStream_t s = (hipStream_t)stream;
    if (grad_x_sorted != nullptr) {
        RowsMm m = input(dtype, ncols_k, nrows_out, n_routes, n_experts, 1);
        m.p = weights, m.q = grad_y, m.y = grad_x_sorted, m.offsets = expert_offsets, m.part = (float *)workspace;
        const hipError_t e = launch_rows_mm(kRowsInput, dtype, m, s);
        if (e != hipSuccess) return launched(e, "mat_mul_rows_grouped_backward input");
    }
    if (grad_weights != nullptr) {
        RowsMm m = weight(dtype, ncols_k, nrows_out, n_routes, n_experts, 1, grad_weights_dtype == JJO_DTYPE_F32);
        m.p = x_sorted, m.q = grad_y, m.y = grad_weights, m.offsets = expert_offsets, m.part = (float *)workspace;
        const hipError_t e = launch_rows_mm(kRowsWeight, dtype, m, s);
        if (e != hipSuccess) return launched(e, "mat_mul_rows_grouped_backward weights");
    }
    return JJO_OK;
}

int64_t moe_rows_gate_up_swiglu_workspace_bytes(int dtype, int hidden_size, int intermediate_size, int n_routes,
                                                int num_experts) {
    clear_error();
    if (check_sizes("moe_rows_gate_up_swiglu", dtype, hidden_size, intermediate_size, n_routes, num_experts) != JJO_OK)
        return -1;
    return rows_part_bytes(kRowsSwiglu, swiglu(dtype, hidden_size, intermediate_size, n_routes, num_experts));
}

int moe_rows_gate_up_swiglu_device(void *stream, const void *x_sorted, const void *w_gate, const void *w_up,
                                   const int32_t *expert_offsets, int num_experts, void *gate_up, void *mid, int dtype,
                                   int hidden_size, int intermediate_size, int n_routes, void *workspace,
                                   int64_t workspace_bytes) {
    clear_error();
    const char *who = "moe_rows_gate_up_swiglu";
    JJO_TRY(check_sizes(who, dtype, hidden_size, intermediate_size, n_routes, num_experts));
    const int es = elem_bytes(dtype);
    JJO_TRY(check_ptr(who, "x_sorted", x_sorted, es));
    JJO_TRY(check_ptr(who, "w_gate", w_gate, es));
    JJO_TRY(check_ptr(who, "w_up", w_up, es));
    JJO_TRY(check_ptr(who, "expert_offsets", expert_offsets, 4));
    JJO_TRY(check_ptr(who, "gate_up", gate_up, es, true));
    JJO_TRY(check_ptr(who, "mid", mid, es));
    RowsMm m = swiglu(dtype, hidden_size, intermediate_size, n_routes, num_experts);
    JJO_TRY(check_workspace(who, workspace, workspace_bytes, rows_part_bytes(kRowsSwiglu, m)));
    JJO_TRY(require_device());
    m.p = w_gate, m.p2 = w_up, m.q = x_sorted, m.y = mid, m.epi.pre = gate_up, m.offsets = expert_offsets;
    m.part = (float *)workspace;
    return launched(launch_rows_mm(kRowsSwiglu, dtype, m, (hipStream_t)stream), "moe_rows_gate_up_swiglu launch");
}

int64_t moe_rows_gate_up_swiglu_backward_workspace_bytes(int dtype, int hidden_size, int intermediate_size,
                                                         int n_routes, int num_experts) {
    clear_error();
    if (check_sizes("moe_rows_gate_up_swiglu_backward", dtype, hidden_size, intermediate_size, n_routes, num_experts) !=
        JJO_OK)
        return -1;
    return swiglu_backward_bytes(dtype, hidden_size, intermediate_size, n_routes, num_experts, gz_planes(dtype), kAll);
}

int64_t moe_rows_gate_up_swiglu_backward_workspace_bytes_for(int dtype, int grad_weights_dtype, int hidden_size,
                                                             int intermediate_size, int n_routes, int num_experts) {
    clear_error();
    const char *who = "moe_rows_gate_up_swiglu_backward";
    if (check_sizes(who, dtype, hidden_size, intermediate_size, n_routes, num_experts) != JJO_OK ||
        check_grad_dtype(who, grad_weights_dtype, dtype) != JJO_OK)
        return -1;
    return swiglu_backward_bytes(dtype, hidden_size, intermediate_size, n_routes, num_experts,
                                 planes_of(dtype, grad_weights_dtype, true, true), kAll);
}

int moe_rows_gate_up_swiglu_backward_device(void *stream, const void *grad_mid, const void *gate_up,
                                            const void *x_sorted, const void *w_gate, const void *w_up,
                                            const int32_t *expert_offsets, int num_experts, void *grad_x_sorted,
                                            void *grad_w_gate, void *grad_w_up, int dtype, int grad_weights_dtype,
                                            int hidden_size, int intermediate_size, int n_routes, void *workspace,
                                            int64_t workspace_bytes) {
    clear_error();
    const char *who = "moe_rows_gate_up_swiglu_backward";
    const int H = hidden_size, I = intermediate_size, R = n_routes, E = num_experts;
    JJO_TRY(check_sizes(who, dtype, H, I, R, E));
    JJO_TRY(check_grad_dtype(who, grad_weights_dtype, dtype));
    const int es = elem_bytes(dtype), ges = elem_bytes(grad_weights_dtype);
    if ((grad_w_gate == nullptr) != (grad_w_up == nullptr))
        return set_error(JJO_ERR_INVALID_ARG, "%s: the gradients of both matrices or of none", who);
    if (grad_x_sorted == nullptr && grad_w_gate == nullptr)
        return set_error(JJO_ERR_INVALID_ARG, "%s: no gradient is asked for", who);
    JJO_TRY(check_ptr(who, "grad_mid", grad_mid, es));
    JJO_TRY(check_ptr(who, "gate_up", gate_up, es));
    JJO_TRY(check_ptr(who, "x_sorted", x_sorted, es, grad_w_gate == nullptr));
    JJO_TRY(check_ptr(who, "w_gate", w_gate, es, grad_x_sorted == nullptr));
    JJO_TRY(check_ptr(who, "w_up", w_up, es, grad_x_sorted == nullptr));
    JJO_TRY(check_ptr(who, "expert_offsets", expert_offsets, 4));
    JJO_TRY(check_ptr(who, "grad_x_sorted", grad_x_sorted, es, true));
    JJO_TRY(check_ptr(who, "grad_w_gate", grad_w_gate, ges, true));
    JJO_TRY(check_ptr(who, "grad_w_up", grad_w_up, ges, true));
    const int planes = planes_of(dtype, grad_weights_dtype, true, grad_w_gate != nullptr);
    JJO_TRY(check_workspace(who, workspace, workspace_bytes,
                            swiglu_backward_bytes(dtype, H, I, R, E, planes,
                                                  {grad_x_sorted != nullptr, grad_w_gate != nullptr, false})));
    JJO_TRY(require_device());
    hipStream_t s = (hipStream_t)stream;
    uint8_t *const gz = (uint8_t *)workspace;
    const int64_t plane = gz_plane_bytes(dtype, 2LL * R * I);
    float *const part = (float *)(gz + planes * plane);
    hipError_t e =
        launch_rows_swiglu_backward(grad_mid, gate_up, gz, planes, plane / es, dtype, expert_offsets, E, I, R, s);
    if (e != hipSuccess) return launched(e, "moe_rows_gate_up_swiglu_backward activation");
    if (grad_x_sorted != nullptr) {
        RowsMm m = input(dtype, H, I, R, E, 2);
        m.p = w_gate, m.p2 = w_up, m.q = gz, m.y = grad_x_sorted, m.offsets = expert_offsets, m.part = part;
        if ((e = launch_rows_mm(kRowsInput, dtype, m, s)) != hipSuccess)
            return launched(e, "moe_rows_gate_up_swiglu_backward input");
    }
    if (grad_w_gate != nullptr) {
        RowsMm m = weight(dtype, H, I, R, E, 2, grad_weights_dtype == JJO_DTYPE_F32);
        m.p = x_sorted, m.y = grad_w_gate, m.y2 = grad_w_up, m.offsets = expert_offsets, m.part = part;
        terms_of_gz(m, gz, plane, planes, es);
        if ((e = launch_rows_mm(kRowsWeight, dtype, m, s)) != hipSuccess)
            return launched(e, "moe_rows_gate_up_swiglu_backward weights");
    }
    return JJO_OK;
}

int jjo_rows_kernel_device(void *stream, int form, int kernel, int slices, int dtype, const void *p, const void *p2,
                           const void *q, const int32_t *expert_offsets, int n_experts, void *y, void *y2, int cols,
                           int rows, int sums, void *workspace, int64_t workspace_bytes) {
    clear_error();
    const char *who = "jjo_rows_kernel";
    JJO_TRY(check_sizes(who, dtype, cols, sums, rows, expert_offsets != nullptr ? n_experts : 1));
    const int es = elem_bytes(dtype), halves = (form == kRowsInput ? (const void *)p2 : y2) != nullptr ? 2 : 1;
    const bool direct = kernel >= 64;
    const int waves = direct ? kernel - 64 : 0;
    if (form < kRowsForward || form > kRowsWeight || slices < 1 || slices > 64 || kernel < 0 ||
        (direct ? form > kRowsSwiglu || slices != 1 || waves < 1 || waves > 8 : kernel >= kRowsTileKinds))
        return set_error(JJO_ERR_INVALID_ARG, "%s: form %d has no kernel %d in %d slices", who, form, kernel, slices);
    JJO_TRY(check_ptr(who, "p", p, es));
    JJO_TRY(check_ptr(who, "p2", p2, es, form != kRowsSwiglu));
    JJO_TRY(check_ptr(who, "q", q, es));
    JJO_TRY(check_ptr(who, "expert_offsets", expert_offsets, 4, true));
    JJO_TRY(check_ptr(who, "y", y, es));
    JJO_TRY(check_ptr(who, "y2", y2, es, true));
    const int E = expert_offsets != nullptr ? n_experts : 0;
    RowsMm m = form == kRowsForward  ? forward(dtype, sums, cols, rows, E)
               : form == kRowsSwiglu ? swiglu(dtype, sums, cols, rows, E)
               : form == kRowsInput  ? input(dtype, cols, sums, rows, E, halves)
                                     : weight(dtype, cols, rows, sums, E, halves, false);
    m.slices = slices;
    JJO_TRY(check_workspace(who, workspace, workspace_bytes, rows_part_bytes((RowsMode)form, m)));
    JJO_TRY(require_device());
    m.p = p, m.p2 = p2, m.q = q, m.y = y, m.y2 = y2, m.offsets = expert_offsets, m.part = (float *)workspace;
    const RowsChoice choice{direct ? (int)kRowsDirect : kernel, waves, slices};
    return launched(launch_rows_mm((RowsMode)form, dtype, m, (hipStream_t)stream, &choice), "jjo_rows_kernel launch");
}

}  // extern "C"
