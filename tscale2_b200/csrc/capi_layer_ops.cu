// extern "C" entry points of include/ts2_b200.h for parts of a training step that the engine does not run: the gated linear
// recurrence, the load balance of a router and its choices, the orthogonalised update, a dense layer, AdamW.
#include "kernels.cuh"

using namespace ts2;

// the calling thread's current device is the caller's again when the call returns
struct OnDevice {
    int before = -1;
    cudaError_t rc;
    explicit OnDevice(int device)
    {
        rc = cudaGetDevice(&before);
        if (rc == cudaSuccess && before != device)
            rc = cudaSetDevice(device);
    }
    ~OnDevice()
    {
        int now = -1;
        if (before >= 0 && cudaGetDevice(&now) == cudaSuccess && now != before)
            cudaSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};
#define TS2_ON_DEVICE(device) \
    OnDevice on_device(device); \
    TS2_CUDA(on_device.rc)

static Ctx layer_ctx(int device, void *stream)
{
    Ctx c;
    c.device = device;
    c.stream = (cudaStream_t)stream;
    return c;
}
// bytes of an element of this type (TS2_OUT_F32, _F16, _BF16), 0: none of them
static int type_size(int type) { return type == TS2_OUT_F32 ? 4 : type == TS2_OUT_F16 || type == TS2_OUT_BF16 ? 2 : 0; }
// a row-major array of at least `cols` columns; without rows it may be null
static bool rows_ok(const void *p, int64_t ld, int64_t rows, int64_t cols, int size)
{
    return (p || rows == 0) && (uintptr_t)p % size == 0 && ld >= cols && ld < ((int64_t)1 << 31);
}
static bool floats_ok(const void *p) { return (uintptr_t)p % 4 == 0; }

// sizes whose tiles can be numbered
static bool linear_sizes_ok(int64_t T, int64_t in_dim, int64_t out_dim)
{
    const int64_t most = (int64_t)1 << 20;
    if (T < 0 || T > (int64_t)1 << 30 || in_dim < 1 || in_dim > most || out_dim < 1 || out_dim > most)
        return false;
    const int64_t dim = in_dim > out_dim ? in_dim : out_dim;
    return ((T + 127) / 128) * ((dim + 63) / 64) < (int64_t)1 << 30;
}
static bool route_sizes_ok(int type, int score, int64_t T, int expert_count, int selected, float scale)
{
    return type_size(type) && (score == TS2_SCORE_SOFTMAX || score == TS2_SCORE_SIGMOID) && T >= 0 && T <= (int64_t)1 << 30 && expert_count >= 1 &&
           selected >= 1 && selected <= expert_count && scale - scale == 0.f;
}

extern "C" {

int ts2_op_recurrence_forward(int device, void *stream, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, int T, int D,
                              int n_seq, const int32_t *seq_ptr, const float *h0, void *h, int64_t h_ld, float *h_last)
{
    const int es = type_size(type);
    if (!es || T < 0 || T > 1 << 30 || D < 1 || D > 65535 * 64 || n_seq < 0 || n_seq > 1 << 30 || (!seq_ptr && n_seq != 1) || !rows_ok(gate, gate_ld, T, D, es) ||
        !rows_ok(x, x_ld, T, D, es) || !rows_ok(h, h_ld, T, D, es) || !floats_ok(seq_ptr) || !floats_ok(h0) || !floats_ok(h_last))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_recurrence_forward: bad arguments");
    TS2_ON_DEVICE(device);
    if (n_seq == 0)
        return TS2_OK;
    return recurrence_forward(layer_ctx(device, stream), type, gate, gate_ld, x, x_ld, T, D, n_seq, seq_ptr, h0, h, h_ld, h_last);
}

int ts2_op_recurrence_backward(int device, void *stream, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, const void *h,
                               int64_t h_ld, int T, int D, int n_seq, const int32_t *seq_ptr, const float *h0, const void *dh, int64_t dh_ld,
                               const float *dh_last, void *dgate, int64_t dgate_ld, void *dx, int64_t dx_ld, float *dh0)
{
    const int es = type_size(type);
    if (!es || T < 0 || T > 1 << 30 || D < 1 || D > 65535 * 64 || n_seq < 0 || n_seq > 1 << 30 || (!seq_ptr && n_seq != 1) || !rows_ok(gate, gate_ld, T, D, es) ||
        !rows_ok(x, x_ld, T, D, es) || !rows_ok(h, h_ld, T, D, es) || !rows_ok(dh, dh_ld, T, D, es) || !rows_ok(dgate, dgate_ld, T, D, es) ||
        !rows_ok(dx, dx_ld, T, D, es) || !floats_ok(seq_ptr) || !floats_ok(h0) || !floats_ok(dh_last) || !floats_ok(dh0))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_recurrence_backward: bad arguments");
    TS2_ON_DEVICE(device);
    if (n_seq == 0)
        return TS2_OK;
    return recurrence_backward(layer_ctx(device, stream), type, gate, gate_ld, x, x_ld, h, h_ld, T, D, n_seq, seq_ptr, h0, dh, dh_ld, dh_last,
                               dgate, dgate_ld, dx, dx_ld, dh0);
}

int ts2_op_moe_balance_forward(int device, void *stream, int type, const void *logits, int64_t ld, int64_t T, int expert_count, int selected,
                               const int32_t *ids, const uint8_t *token_mask, int32_t *counts, float *prob, float *loss)
{
    const int es = type_size(type);
    if (!es || T < 0 || T > 1 << 30 || expert_count < 1 || selected < 1 || selected > expert_count || T * selected >= (int64_t)1 << 31 ||
        !rows_ok(logits, ld, T, expert_count, es) || (!ids && T) || !floats_ok(ids) || !counts || !prob || !loss || !floats_ok(counts) ||
        !floats_ok(prob) || !floats_ok(loss))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_moe_balance_forward: bad arguments");
    if (expert_count > MOE_BALANCE_MAX_EXPERTS)
        return fail(TS2_ERR_UNSUPPORTED, "ts2_op_moe_balance_forward: at most %d experts (got %d)", MOE_BALANCE_MAX_EXPERTS, expert_count);
    TS2_ON_DEVICE(device);
    return moe_balance_forward(layer_ctx(device, stream), type, logits, ld, T, expert_count, selected, ids, token_mask, counts, prob, loss);
}

int ts2_op_moe_balance_backward(int device, void *stream, int type, const void *logits, int64_t ld, int64_t T, int expert_count, int selected,
                                const uint8_t *token_mask, const int32_t *counts, const float *dloss, float scale, void *dlogits, int64_t dlogits_ld,
                                int add)
{
    const int es = type_size(type);
    if (!es || T < 0 || T > 1 << 30 || expert_count < 1 || selected < 1 || selected > expert_count || !rows_ok(logits, ld, T, expert_count, es) || !counts ||
        !floats_ok(counts) || !floats_ok(dloss) || !rows_ok(dlogits, dlogits_ld, T, expert_count, es))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_moe_balance_backward: bad arguments");
    if (expert_count > MOE_BALANCE_MAX_EXPERTS)
        return fail(TS2_ERR_UNSUPPORTED, "ts2_op_moe_balance_backward: at most %d experts (got %d)", MOE_BALANCE_MAX_EXPERTS, expert_count);
    TS2_ON_DEVICE(device);
    return moe_balance_backward(layer_ctx(device, stream), type, logits, ld, T, expert_count, selected, token_mask, counts, dloss, scale, dlogits,
                                dlogits_ld, add != 0);
}

int ts2_op_orthogonalize(int device, void *stream, int type, const void *g, int64_t ld, int64_t g_stride, int batch, int64_t rows, int64_t cols,
                         const float coef[3], int steps, float out_scale, void *out, int64_t out_ld, int64_t out_stride)
{
    const int es = type_size(type);
    if (!es || batch < 0 || batch > 65535 || rows < 1 || cols < 1 || rows > 1 << 20 || cols > 1 << 20 || !coef || steps < 1 || steps > 64 ||
        g_stride < 0 || !rows_ok(g, ld, batch, cols, es) || !rows_ok(out, out_ld, batch, cols, 2) ||
        (batch > 1 && out_stride < (rows - 1) * out_ld + cols))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_orthogonalize: bad arguments");
    if (!orthogonalize_in_range(coef, steps))
        return fail(TS2_ERR_UNSUPPORTED, "ts2_op_orthogonalize: the coefficients take singular values out of the range of fp16");
    TS2_ON_DEVICE(device);
    if (batch == 0)
        return TS2_OK;
    return orthogonalize(layer_ctx(device, stream), type, g, ld, g_stride, batch, (int)rows, (int)cols, coef, steps, out_scale, out, out_ld,
                         out_stride);
}

int ts2_op_linear_forward(int device, void *stream, int type, int act, int64_t T, int64_t in_dim, int64_t out_dim, const void *x, int64_t x_ld,
                          const void *w, int64_t w_ld, const float *bias, const void *residual, int64_t residual_ld, void *y, int64_t y_ld, void *z,
                          int64_t z_ld)
{
    if ((type != TS2_OUT_F16 && type != TS2_OUT_BF16) || act < TS2_ACT_NONE || act > TS2_ACT_SILU || !linear_sizes_ok(T, in_dim, out_dim) ||
        !rows_ok(x, x_ld, T, in_dim, 2) || !rows_ok(w, w_ld, out_dim, in_dim, 2) || !floats_ok(bias) || !rows_ok(y, y_ld, T, out_dim, 2) ||
        (residual && (!rows_ok(residual, residual_ld, T, out_dim, 2) || (residual == y && residual_ld != y_ld))) ||
        (z && !rows_ok(z, z_ld, T, out_dim, 2)))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_linear_forward: bad arguments");
    TS2_ON_DEVICE(device);
    const LinearShape s = {T, (int)in_dim, (int)out_dim, type, act};
    return linear_forward(layer_ctx(device, stream), s, x, x_ld, w, w_ld, bias, residual, residual_ld, y, y_ld, z, z_ld);
}

int ts2_op_linear_backward(int device, void *stream, int type, int act, int64_t T, int64_t in_dim, int64_t out_dim, const void *dy, int64_t dy_ld,
                           const void *z, int64_t z_ld, const void *x, int64_t x_ld, const void *w, int64_t w_ld, void *dx, int64_t dx_ld,
                           int dw_kind, void *dw, int64_t dw_ld, float *dbias)
{
    const bool kind_ok = dw_kind == type || dw_kind == TS2_OUT_F32 || dw_kind == TS2_OUT_F32_ADD;
    if ((type != TS2_OUT_F16 && type != TS2_OUT_BF16) || act < TS2_ACT_NONE || act > TS2_ACT_SILU || !linear_sizes_ok(T, in_dim, out_dim) ||
        !rows_ok(dy, dy_ld, T, out_dim, 2) || (act != TS2_ACT_NONE && !rows_ok(z, z_ld, T, out_dim, 2)) ||
        (dw && (!kind_ok || !rows_ok(x, x_ld, T, in_dim, 2) || !rows_ok(dw, dw_ld, out_dim, in_dim, dw_kind == type ? 2 : 4))) ||
        (dx && (!rows_ok(w, w_ld, out_dim, in_dim, 2) || !rows_ok(dx, dx_ld, T, in_dim, 2))) || !floats_ok(dbias))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_linear_backward: bad arguments");
    TS2_ON_DEVICE(device);
    const LinearShape s = {T, (int)in_dim, (int)out_dim, type, act};
    return linear_backward(layer_ctx(device, stream), s, dy, dy_ld, z, z_ld, x, x_ld, w, w_ld, dx, dx_ld, dw_kind, dw, dw_ld, dbias);
}

int ts2_op_moe_route_forward(int device, void *stream, int type, int score, const void *logits, int64_t ld, int64_t T, int expert_count, int selected,
                             const float *bias, int groups, int groups_kept, int group_top, int renormalize, float scale, const uint8_t *token_mask,
                             int32_t *ids, float *weights)
{
    if (!route_sizes_ok(type, score, T, expert_count, selected, scale) || !rows_ok(logits, ld, T, expert_count, type_size(type)) || !floats_ok(bias) ||
        groups < 1 || groups > expert_count || expert_count % groups || groups_kept < 1 || groups_kept > groups || group_top < 1 || group_top > 2 ||
        group_top > expert_count / groups || (int64_t)selected * groups > (int64_t)expert_count * groups_kept || (T && (!ids || !weights)) ||
        !floats_ok(ids) || !floats_ok(weights))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_moe_route_forward: bad arguments");
    if (expert_count > MOE_ROUTE_MAX_EXPERTS || selected > MOE_ROUTE_MAX_SELECTED || groups > MOE_ROUTE_MAX_GROUPS)
        return fail(TS2_ERR_UNSUPPORTED, "ts2_op_moe_route_forward: at most %d experts, %d of them selected, in %d groups (got %d, %d, %d)",
                    MOE_ROUTE_MAX_EXPERTS, MOE_ROUTE_MAX_SELECTED, MOE_ROUTE_MAX_GROUPS, expert_count, selected, groups);
    TS2_ON_DEVICE(device);
    const RouteShape s = {type, score, T, expert_count, selected, renormalize != 0, scale};
    return moe_route_forward(layer_ctx(device, stream), s, logits, ld, bias, groups, groups_kept, group_top, token_mask, ids, weights);
}

int ts2_op_moe_route_backward(int device, void *stream, int type, int score, const void *logits, int64_t ld, int64_t T, int expert_count, int selected,
                              int renormalize, float scale, const uint8_t *token_mask, const int32_t *ids, const float *dweights, void *dlogits,
                              int64_t dlogits_ld, int add)
{
    const int es = type_size(type);
    if (!route_sizes_ok(type, score, T, expert_count, selected, scale) || !rows_ok(logits, ld, T, expert_count, es) || (T && (!ids || !dweights)) ||
        !floats_ok(ids) || !floats_ok(dweights) || !rows_ok(dlogits, dlogits_ld, T, expert_count, es))
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_moe_route_backward: bad arguments");
    if (expert_count > MOE_ROUTE_MAX_EXPERTS || selected > MOE_ROUTE_MAX_SELECTED)
        return fail(TS2_ERR_UNSUPPORTED, "ts2_op_moe_route_backward: at most %d experts, %d of them selected (got %d, %d)", MOE_ROUTE_MAX_EXPERTS,
                    MOE_ROUTE_MAX_SELECTED, expert_count, selected);
    TS2_ON_DEVICE(device);
    const RouteShape s = {type, score, T, expert_count, selected, renormalize != 0, scale};
    return moe_route_backward(layer_ctx(device, stream), s, logits, ld, token_mask, ids, dweights, dlogits, dlogits_ld, add != 0);
}

int ts2_op_adamw(int device, void *stream, int grad_type, int state_bits, int copy_type, const ts2_adamw_tensor *tensors, int n_tensors, float rate,
                 float beta1, float beta2, float eps, int64_t step, float grad_scale, const float *grad_scale_dev, uint64_t seed)
{
    const auto finite = [](float v) { return v - v == 0.f; };
    bool ok = type_size(grad_type) && (state_bits == 32 || state_bits == 8) && type_size(copy_type) && n_tensors >= 0 && n_tensors <= 1 << 20 &&
              (tensors || !n_tensors) && finite(rate) && beta1 >= 0.f && beta1 < 1.f && beta2 >= 0.f && beta2 < 1.f && eps >= 0x1p-126f && finite(eps) && step >= 1 &&
              finite(grad_scale) && floats_ok(grad_scale_dev);
    int64_t total = 0;
    for (int i = 0; ok && i < n_tensors; ++i) {
        const ts2_adamw_tensor &t = tensors[i];
        const auto array = [&](const void *p, int size) { return (p || t.n == 0) && (uintptr_t)p % size == 0; };
        ok = t.n >= 0 && t.n <= (int64_t)1 << 40 && array(t.param, 4) && array(t.grad, type_size(grad_type)) && array(t.m, state_bits / 8) &&
             array(t.v, state_bits / 8) && (state_bits == 32 || (array(t.m_scale, 1) && array(t.v_scale, 1))) &&
             (!t.copy || (copy_type != TS2_OUT_F32 && array(t.copy, 2))) && finite(t.rate) && finite(t.decay);
        total += ok ? t.n : 0;
        ok = ok && total <= (int64_t)1 << 40;
    }
    if (!ok)
        return fail(TS2_ERR_INVALID_ARG, "ts2_op_adamw: bad arguments");
    TS2_ON_DEVICE(device);
    return adamw(layer_ctx(device, stream), grad_type, state_bits, copy_type, tensors, n_tensors, rate, beta1, beta2, eps, step, grad_scale,
                 grad_scale_dev, seed);
}

} // extern "C"
