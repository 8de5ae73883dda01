// extern "C" entry points of include/ts2_b200.h for parts of a training step that the engine does not run: the gated linear
// recurrence, the load balance of a router, the orthogonalised update.
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

} // extern "C"
