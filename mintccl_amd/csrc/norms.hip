// Norms and the residual stream (norms.hpp): the sums over rows joined, and the entry points.
#include "norms.hpp"

namespace mint {
namespace {

// ---- the sums over rows, joined ----------------------------------------------------
struct ColumnSumsArgs {
    const float* sums;                          // (groups, n, width)
    void *before_weight, *before_bias, *after_weight, *after_bias, *to_gate;      // any may be 0
    const void* gate;                           // by channel, or 0
    NormArgs before, after;
    uint32_t groups, width, n;
    int gate_dtype, gate_by;
    bool block, bias;
};
// A thread block has 16 columns, and 16 lanes every 64th group's sums of them.  512 groups of two sums of 4096: 6 us.
constexpr int kColumnWaves = 16;
__global__ void __launch_bounds__(64 * kColumnWaves) column_sums_kernel(ColumnSumsArgs a) {
    __shared__ float part[4][kColumnWaves * 4][16];
    const uint32_t lane = threadIdx.x & 15u, slot = threadIdx.x >> 4, col = block_in_grid() * 16 + lane, from = min(col, a.width - 1);
    constexpr uint32_t SLOTS = kColumnWaves * 4;
    for (uint32_t k = 0; k < a.n; ++k) {
        float sum = 0.0f;
        for (uint32_t g0 = slot; g0 < a.groups; g0 += SLOTS * 8) {
            float v[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) v[u] = *as_global(a.sums + ((uint64_t)min(g0 + u * SLOTS, a.groups - 1) * a.n + k) * a.width + from);
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) sum += g0 + u * SLOTS < a.groups ? v[u] : 0.0f;
        }
        part[k][slot][lane] = sum;
    }
    __syncthreads();
    // 64 slots, 16 at a time
    if (slot < 4) {
        for (uint32_t k = 0; k < a.n; ++k) {
            float sum = 0.0f;
#pragma unroll
            for (uint32_t u = 0; u < 16; ++u) sum += part[k][slot * 16 + u][lane];
            part[k][slot * 16][lane] = sum;
        }
    }
    __syncthreads();
    if (slot != 0 || col >= a.width) return;
    float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
        if (k < a.n) total[k] = (part[k][0][lane] + part[k][16][lane]) + (part[k][32][lane] + part[k][48][lane]);
    if (a.before_weight) store_one(a.before_weight, a.before.dtype, col, total[0]);
    if (a.before_bias) store_one(a.before_bias, a.before.dtype, col, total[1]);
    if (!a.block) return;
    const float of_w = a.bias ? total[2] : total[1], of_b = total[3];
    const float raw = a.gate ? load_one(a.gate, a.gate_dtype, col) : 0.0f, open = a.gate ? gate_value(a.gate_by, raw) : 1.0f;
    if (a.after_weight) store_one(a.after_weight, a.after.dtype, col, open * of_w);
    if (a.after_bias) store_one(a.after_bias, a.after.dtype, col, open * of_b);
    if (a.to_gate) {
        const float w = a.after.weight ? load_one(a.after.weight, a.after.dtype, col) : 1.0f;
        const float b = a.after.bias ? load_one(a.after.bias, a.after.dtype, col) : 0.0f;
        store_one(a.to_gate, a.gate_dtype, col, gate_slope(a.gate_by, raw) * (b == 0.0f ? w * of_w : fmaf(w, of_w, b * of_b)));
    }
}

// The gradients of gates by row whose rows have no numbers: sums of nothing.
__global__ void __launch_bounds__(256) clear_gates_kernel(void* to_gate, int dtype, int64_t stride, uint32_t rows) {
    const uint32_t r = blockIdx.x * 256 + threadIdx.x;
    if (r < rows) store_one(to_gate, dtype, (int64_t)r * stride, 0.0f);
}

// ---- the entry points --------------------------------------------------------------
// the types that go together: the stream is of the block's type, or in 32 bits
#define MINT_STREAM_TYPES(GO, ...)                                                                                          \
    switch (op->dtype) {                                                                                                    \
        case MINT_F16: return op->stream_dtype == MINT_F16 ? GO##_f16(__VA_ARGS__) : GO##_f32_f16(__VA_ARGS__);             \
        case MINT_BF16: return op->stream_dtype == MINT_BF16 ? GO##_bf16(__VA_ARGS__) : GO##_f32_bf16(__VA_ARGS__);         \
        default: return GO##_f32(__VA_ARGS__);                                                                              \
    }

bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }
bool norm_known(const mint_norm& n, bool may_be_none) {
    if (n.kind == MINT_NORM_NONE) return may_be_none && !n.weight && !n.bias;
    return (n.kind == MINT_NORM_RMS || n.kind == MINT_NORM_LAYER) && ((!n.weight && !n.bias) || known(n.dtype));
}
NormArgs norm_args(const mint_norm& n) {
    return {reinterpret_cast<const void*>(n.weight), reinterpret_cast<const void*>(n.bias), n.kind, n.dtype, n.eps};
}
int join_args(const mint_join_op* op, JoinArgs& a) {
    if (!op || !known(op->dtype) || !(op->stream_dtype == op->dtype || op->stream_dtype == MINT_F32) || !gate_known(op->gate_by) ||
        !norm_known(op->before, true) || !norm_known(op->after, true))
        return MINT_ERR_ARG;
    if (op->gate && (!known(op->gate_dtype) || op->gate_form < MINT_GATE_CHANNEL || op->gate_form > MINT_GATE_ALL)) return MINT_ERR_ARG;
    if (op->rows && op->width && !op->y && (op->gate || op->after.kind)) return MINT_ERR_ARG;
    if (op->rows > 0x7FFFFFFF / 4 || op->width > 0x7FFFFFFF - kLongThreads * V) return MINT_ERR_TOO_LARGE;
    a = {reinterpret_cast<const void*>(op->stream), reinterpret_cast<const void*>(op->y), reinterpret_cast<const void*>(op->gate),
         reinterpret_cast<void*>(op->new_stream), reinterpret_cast<void*>(op->next),
         op->stream_stride, op->y_stride, op->gate_row, op->new_stride, op->next_stride, norm_args(op->after), norm_args(op->before), op->scale, op->carry,
         (uint32_t)op->rows, (uint32_t)op->width, op->gate_dtype, op->gate_by, op->gate_form};
    if (op->gate_form == MINT_GATE_CHANNEL) a.gate_row = 0;
    return MINT_OK;
}

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" int mint_join(const mint_join_op* op, void* stream) {
    JoinArgs a;
    if (const int err = join_args(op, a)) return err;
    if (a.rows == 0 || a.width == 0) return MINT_OK;
    if (!a.stream || (a.y && !a.new_stream) || (a.next && !a.before.kind) || (!a.y && !a.next)) return MINT_ERR_ARG;
    if (a.width > kLongest && (uint64_t)a.rows * a.width > 1ull << 40) return MINT_ERR_TOO_LARGE;      // (no memory holds the results)
    const auto s = static_cast<hipStream_t>(stream);
    MINT_STREAM_TYPES(launch_join, a, s)
}

namespace {
bool grad_bias(const mint_join_op& f) { return f.before.bias || f.after.bias; }
bool grad_sums(const mint_join_grad_op& op) {
    return op.to_before_weight || op.to_before_bias || op.to_after_weight || op.to_after_bias ||
           (op.to_gate && op.join.gate_form == MINT_GATE_CHANNEL);
}
uint64_t grad_workspace(const mint_join_grad_op& op) {
    if (!grad_sums(op) || op.join.rows == 0) return 0;
    const uint64_t n = (op.join.y ? 2 : 1) * (grad_bias(op.join) ? 2 : 1);
    return blocks_of(op.join.rows, op.join.width) * n * op.join.width * 4;
}
}  // namespace

extern "C" size_t mint_join_grad_workspace(const mint_join_grad_op* op) { return op ? grad_workspace(*op) : 0; }

extern "C" int mint_join_grad(const mint_join_grad_op* op_grad, void* stream) {
    if (!op_grad) return MINT_ERR_ARG;
    const mint_join_op* const op = &op_grad->join;
    JoinGradArgs a = {};
    if (const int err = join_args(op, a.f)) return err;
    if (a.f.width == 0) {
        if (!op_grad->to_gate || !a.f.gate || op->gate_form != MINT_GATE_ROW || a.f.rows == 0) return MINT_OK;
        return Launch<&clear_gates_kernel>::go((a.f.rows + 255) / 256, 256, 0, static_cast<hipStream_t>(stream), reinterpret_cast<void*>(op_grad->to_gate),
                                               op->gate_dtype, op_grad->to_gate_stride, a.f.rows);
    }
    if (op_grad->to_gate && !a.f.gate) return MINT_ERR_ARG;
    if ((op_grad->to_y || op_grad->to_after_weight || op_grad->to_after_bias) && !a.f.y && a.f.rows) return MINT_ERR_ARG;
    if ((op_grad->to_before_weight && !op->before.weight) || (op_grad->to_before_bias && !op->before.bias) ||
        (op_grad->to_after_weight && !op->after.weight) || (op_grad->to_after_bias && !op->after.bias))
        return MINT_ERR_ARG;
    if (a.f.rows && (op_grad->d_next ? !a.f.stream || !a.f.before.kind : !op_grad->d_stream)) return MINT_ERR_ARG;
    const uint64_t need = grad_workspace(*op_grad);
    if (need && (!op_grad->workspace || op_grad->workspace_bytes < need)) return MINT_ERR_STAGING;
    if (need && op_grad->workspace % 4) return MINT_ERR_ALIGN;
    a.d_stream = reinterpret_cast<const void*>(op_grad->d_stream);
    a.d_next = reinterpret_cast<const void*>(op_grad->d_next);
    a.to_stream = reinterpret_cast<void*>(op_grad->to_stream);
    a.to_y = reinterpret_cast<void*>(op_grad->to_y);
    a.to_gate = reinterpret_cast<void*>(op_grad->to_gate);
    a.d_stream_stride = op_grad->d_stream_stride;
    a.d_next_stride = op_grad->d_next_stride;
    a.to_stream_stride = op_grad->to_stream_stride;
    a.to_y_stride = op_grad->to_y_stride;
    a.to_gate_stride = op_grad->to_gate_stride;
    a.sums = need ? reinterpret_cast<float*>(op_grad->workspace) : nullptr;
    a.groups = blocks_of(a.f.rows, a.f.width);
    const bool bias = grad_bias(*op), by_channel = a.f.gate && a.f.gate_form == MINT_GATE_CHANNEL;
    const auto s = static_cast<hipStream_t>(stream);
    const auto rows = [&]() -> int { MINT_STREAM_TYPES(launch_join_grad, a, bias, s) };
    if (a.f.rows) {
        const int err = rows();
        if (err != MINT_OK) return err;
    }
    if (!grad_sums(*op_grad)) return MINT_OK;
    // (of no rows the sums are zeros)
    const ColumnSumsArgs c = {a.sums, reinterpret_cast<void*>(op_grad->to_before_weight), reinterpret_cast<void*>(op_grad->to_before_bias),
                              reinterpret_cast<void*>(op_grad->to_after_weight), reinterpret_cast<void*>(op_grad->to_after_bias),
                              by_channel ? a.to_gate : nullptr, by_channel ? a.f.gate : nullptr, a.f.before, a.f.after, a.f.rows ? a.groups : 0u, a.f.width,
                              a.f.rows ? (a.f.y ? 2u : 1u) * (bias ? 2u : 1u) : 0u, a.f.gate_dtype, a.f.gate_by, a.f.y != nullptr || !a.f.rows, bias};
    return Launch<&column_sums_kernel>::go(wide_grid(ceil_div(a.f.width, 16)), 64 * kColumnWaves, 0, s, c);
}
