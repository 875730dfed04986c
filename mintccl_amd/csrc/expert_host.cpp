// mintccl_amd._expert_host: the host side of the operators of an expert layer (routing.py, block8.py,
// combine.py) and around it (norms.py, dense.py), native: a call for one token takes the GPU a few us, and so must the checks of
// its arguments, its outputs' allocation and the launch.  What a call allocates for itself
// comes from torch's allocator on the calling thread's current stream, on which it launches too.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <stdexcept>

#include "../../include/mintccl.h"

namespace {

struct Native {
    decltype(&mint_route) route;
    decltype(&mint_route_grad) route_grad;
    decltype(&mint_assign_workspace) assign_workspace;
    decltype(&mint_assign) assign;
    decltype(&mint_rows8) rows8;
    decltype(&mint_squares8) squares8;
    decltype(&mint_product8_workspace) product8_workspace;
    decltype(&mint_product8) product8;
    decltype(&mint_weight_grad8_workspace) weight_grad8_workspace;
    decltype(&mint_weight_grad8) weight_grad8;
    decltype(&mint_combine) combine;
    decltype(&mint_combine_grad) combine_grad;
    decltype(&mint_join) join;
    decltype(&mint_join_grad_workspace) join_grad_workspace;
    decltype(&mint_join_grad) join_grad;
    decltype(&mint_dense_workspace) dense_workspace;
    decltype(&mint_dense) dense;
    decltype(&mint_activation_grad_workspace) activation_grad_workspace;
    decltype(&mint_activation_grad) activation_grad;
    decltype(&mint_balance_workspace) balance_workspace;
    decltype(&mint_balance) balance;
    decltype(&mint_balance_grad) balance_grad;
    PyObject* check;             // _lib.check(code, where): raises MintError
} native = {};

using at::Tensor;

// A refusal: its Python type and text.
struct Refused : std::exception {
    PyObject* type;
    char text[256];
    const char* what() const noexcept override { return text; }
};
[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    Refused r;
    r.type = type;
    va_list list;
    va_start(list, format);
    vsnprintf(r.text, sizeof(r.text), format, list);
    va_end(list);
    throw r;
}
struct Raised {};                // a Python exception is set

template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Raised&) {
        return nullptr;
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.text);
    } catch (const std::bad_alloc&) {
        return PyErr_NoMemory();
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
void checked(int code, const char* where) {
    if (code == MINT_OK) return;
    PyObject* r = PyObject_CallFunction(native.check, "is", code, where);
    Py_XDECREF(r);
    throw Raised();
}

// The current device is the operands' for as long as this lives; `stream` is its current one.
struct OnDevice {
    int before, device;
    void* stream;
    explicit OnDevice(int d) : before(only() ? d : (int)c10::hip::current_device()), device(d) {
        if (before != device) c10::hip::set_device((c10::DeviceIndex)device);
        const auto current = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device);
        stream = current.id() == 0 ? nullptr : (void*)current.stream();
    }
    static bool only() {
        static const bool one = c10::hip::device_count() == 1;
        return one;
    }
    ~OnDevice() {
        if (before != device) c10::hip::set_device((c10::DeviceIndex)before);
    }
};

// Launches may wait for the device's queue: other Python threads go on meanwhile.
template <typename F>
void launch(const char* where, F&& f) {
    int code;
    Py_BEGIN_ALLOW_THREADS
    code = f();
    Py_END_ALLOW_THREADS
    checked(code, where);
}

// ---- arguments -----------------------------------------------------------------
struct Args {
    PyObject* const* list;
    Args(PyObject* const* a, Py_ssize_t n, Py_ssize_t wanted) : list(a) {
        if (n != wanted) refuse(PyExc_TypeError, "%zd arguments are wanted", wanted);
    }
    bool none(int i) const { return list[i] == Py_None; }
    // `history`: whether the results have a gradient by it
    const Tensor& tensor(int i, const char* name, bool history = true) const {
        if (!THPVariable_Check(list[i])) refuse(PyExc_TypeError, "%s must be a device tensor", name);
        const Tensor& t = THPVariable_Unpack(list[i]);
        if (!t.is_cuda() || t.layout() != at::kStrided) refuse(PyExc_TypeError, "%s must be a device tensor", name);
        // (a result without a history, or without a tangent, would end the gradient here without a word)
        if (history && t.requires_grad() && c10::GradMode::is_enabled())
            refuse(PyExc_RuntimeError, "%s requires a gradient, and these operators record none: detach it, or call under torch.no_grad()", name);
        if (history && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
            refuse(PyExc_RuntimeError, "%s has a tangent, and these operators hand none on: unpack it, or call under torch.inference_mode()", name);
        return t;
    }
    int64_t integer(int i, const char* name, int64_t least, int64_t most) const {
        PyObject* index = PyNumber_Index(list[i]);
        if (!index) throw Raised();
        int over = 0;
        const long long v = PyLong_AsLongLongAndOverflow(index, &over);
        Py_DECREF(index);
        if (over || v < least || v > most) refuse(PyExc_ValueError, "%s must be in %lld..%lld", name, (long long)least, (long long)most);
        return v;
    }
    bool truth(int i) const {
        const int v = PyObject_IsTrue(list[i]);
        if (v < 0) throw Raised();
        return v;
    }
    float number(int i) const {
        const double v = PyFloat_AsDouble(list[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Raised();
        return (float)v;
    }
};

int code_of(at::ScalarType t, const char* name) {
    switch (t) {
        case at::kHalf: return MINT_F16;
        case at::kBFloat16: return MINT_BF16;
        case at::kFloat: return MINT_F32;
        default: refuse(PyExc_TypeError, "%s must be float16, bfloat16 or float32", name);
    }
}
at::ScalarType type_of(int64_t code) {
    return code == MINT_F16 ? at::kHalf : code == MINT_BF16 ? at::kBFloat16 : at::kFloat;
}
void same_device(const Tensor& a, const Tensor& b, const char* name) {
    if (a.get_device() != b.get_device()) refuse(PyExc_ValueError, "%s lives on another device", name);
}
void dims(const Tensor& t, int64_t n, const char* name) {
    if (t.dim() != n) refuse(PyExc_ValueError, "%s must have %lld dimensions", name, (long long)n);
}
// rows whose numbers lie side by side, any distance apart
void rows_of(const Tensor& t, const char* name) {
    dims(t, 2, name);
    if (t.size(1) > 1 && t.stride(1) != 1) refuse(PyExc_ValueError, "the rows of %s must lie in one piece each", name);
}
void typed(const Tensor& t, at::ScalarType type, const char* name, const char* what) {
    if (t.scalar_type() != type) refuse(PyExc_TypeError, "%s must be %s", name, what);
}
void dense(const Tensor& t, const char* name) {
    if (!t.is_contiguous()) refuse(PyExc_ValueError, "%s must be contiguous", name);
}
// a result that the caller brings: rows that do not overlap
void result(const Tensor& t, int64_t rows, int64_t cols, const char* name) {
    rows_of(t, name);
    if (t.size(0) != rows || t.size(1) != cols)
        refuse(PyExc_ValueError, "%s must be (%lld, %lld)", name, (long long)rows, (long long)cols);
    if (rows > 1 && cols > 0 && t.stride(0) < cols) refuse(PyExc_ValueError, "the rows of %s overlap", name);
}
// ... and that none of the call's rows or vectors lie in, but for one that may be the result itself.  (Rows of one buffer side by side may.)
void clear_of(const Tensor& out, const Tensor& t, const char* name, bool may_be_it) {
    if (out.numel() == 0 || t.numel() == 0 || out.get_device() != t.get_device()) return;
    const auto row = [](const Tensor& x) { return (uint64_t)(x.size(-1) * (int64_t)x.element_size()); };
    const auto pitch = [](const Tensor& x) { return x.dim() > 1 && x.size(0) > 1 ? (uint64_t)(x.stride(0) * (int64_t)x.element_size()) : 0; };
    const uint64_t p = (uint64_t)out.data_ptr(), q = (uint64_t)t.data_ptr(), every = pitch(out), also = pitch(t);
    if (p + (every ? every * (out.size(0) - 1) : 0) + row(out) <= q || q + (also ? also * (t.size(0) - 1) : 0) + row(t) <= p) return;
    if (may_be_it && p == q && every == also && out.scalar_type() == t.scalar_type()) return;
    if (every && every == also) {
        const uint64_t behind = q >= p ? (q - p) % every : (every - (p - q) % every) % every;
        if (behind >= row(out) && behind + row(t) <= every) return;
    }
    refuse(PyExc_ValueError, "out shares memory with %s", name);
}
Tensor empty(const Tensor& like, at::IntArrayRef size, at::ScalarType type) {
    return at::empty(size, at::TensorOptions().device(like.device()).dtype(type));
}
// (detached from `like`'s type and layout: only its device counts)
PyObject* wrap(const Tensor& t) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) throw Raised();
    return o;
}
PyObject* pack(std::initializer_list<PyObject*> list) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)list.size());
    Py_ssize_t i = 0;
    for (PyObject* o : list) {
        if (tuple) PyTuple_SET_ITEM(tuple, i++, o);
        else Py_DECREF(o);
    }
    if (!tuple) throw Raised();
    return tuple;
}
uint64_t address(const Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }

// ---- routing -------------------------------------------------------------------
// route(logits, topk, score, bias, groups, kept, group_top, renormalise, scale)
PyObject* host_route(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 9);
        const Tensor& x = a.tensor(0, "logits");
        rows_of(x, "logits");
        mint_route_op op = {};
        op.dtype = code_of(x.scalar_type(), "logits");
        op.tokens = (uint64_t)x.size(0);
        op.experts = (uint32_t)std::min<int64_t>(x.size(1), 1u << 30);
        if (x.size(1) < 1 || x.size(1) > 1024) refuse(PyExc_ValueError, "logits must be of 1..1024 experts");
        op.topk = (uint32_t)a.integer(1, "k", 1, std::min<int64_t>(64, x.size(1)));
        op.score = (int32_t)a.integer(2, "score", 0, 1);
        op.groups = (uint32_t)a.integer(4, "groups", 1, 64);
        if (x.size(1) % op.groups) refuse(PyExc_ValueError, "the experts do not divide into %u groups", op.groups);
        op.kept = (uint32_t)a.integer(5, "kept", 1, op.groups);
        op.group_top = (uint32_t)a.integer(6, "group_top", 1, 2);
        op.renormalise = a.truth(7);
        op.scale = a.number(8);
        op.logits = address(x);
        op.row_stride = x.stride(0);
        if (!a.none(3)) {
            const Tensor& bias = a.tensor(3, "bias", false);
            same_device(x, bias, "bias");
            typed(bias, at::kFloat, "bias", "float32");
            dims(bias, 1, "bias");
            dense(bias, "bias");
            if (bias.size(0) != x.size(1)) refuse(PyExc_ValueError, "bias must have a number for each expert");
            op.bias = address(bias);
        }
        OnDevice on(x.get_device());
        const Tensor weights = empty(x, {x.size(0), (int64_t)op.topk}, at::kFloat), chosen = empty(x, {x.size(0), (int64_t)op.topk}, at::kInt);
        op.weights = address(weights);
        op.chosen = address(chosen);
        launch("mint_route", [&] { return native.route(&op, on.stream); });
        return pack({wrap(weights), wrap(chosen)});
    });
}

// (tokens, k) int32, contiguous
void choices(const Tensor& t, const char* name) {
    dims(t, 2, name);
    typed(t, at::kInt, name, "int32");
    dense(t, name);
    if (t.size(1) < 1) refuse(PyExc_ValueError, "%s must have a column at least", name);
}
void weights_of(const Tensor& w, const Tensor& like, const char* name) {
    same_device(like, w, name);
    dims(w, 2, name);
    typed(w, at::kFloat, name, "float32");
    dense(w, name);
    if (w.sizes() != like.sizes()) refuse(PyExc_ValueError, "%s must have a number for each choice", name);
}

// route_grad(d_weights, logits, experts, score, renormalise, scale)
PyObject* host_route_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 6);
        const Tensor &d = a.tensor(0, "grad"), &x = a.tensor(1, "logits"), &chosen = a.tensor(2, "experts");
        rows_of(x, "logits");
        same_device(x, chosen, "experts");
        choices(chosen, "experts");
        weights_of(d, chosen, "grad");
        if (x.size(1) < 1 || x.size(1) > 1024) refuse(PyExc_ValueError, "logits must be of 1..1024 experts");
        if (chosen.size(0) != x.size(0) || chosen.size(1) > std::min<int64_t>(64, x.size(1)))
            refuse(PyExc_ValueError, "experts must be what was chosen by these logits");
        mint_route_op op = {};
        op.dtype = code_of(x.scalar_type(), "logits");
        op.tokens = (uint64_t)x.size(0);
        op.experts = (uint32_t)x.size(1);
        op.topk = (uint32_t)chosen.size(1);
        op.score = (int32_t)a.integer(3, "score", 0, 1);
        op.renormalise = a.truth(4);
        op.scale = a.number(5);
        op.logits = address(x);
        op.row_stride = x.stride(0);
        op.chosen = address(chosen);
        OnDevice on(x.get_device());
        const Tensor out = empty(x, x.sizes(), x.scalar_type());
        launch("mint_route_grad", [&] { return native.route_grad(&op, address(d), address(out), out.stride(0), on.stream); });
        return wrap(out);
    });
}

// assign(experts, count, first)
PyObject* host_assign(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 3);
        const Tensor& chosen = a.tensor(0, "experts");
        choices(chosen, "experts");
        const int64_t count = a.integer(1, "count", 1, 1024), first = a.integer(2, "first", 0, 0x7FFFFFFF - 1024);
        const int64_t pairs = chosen.numel();
        OnDevice on(chosen.get_device());
        const Tensor offsets = empty(chosen, {count + 1}, at::kInt), order = empty(chosen, {pairs}, at::kInt), slots = empty(chosen, chosen.sizes(), at::kInt);
        const size_t need = native.assign_workspace((uint64_t)pairs, (uint32_t)count);
        Tensor room;
        if (need) room = empty(chosen, {(int64_t)need}, at::kByte);
        launch("mint_assign", [&] {
            return native.assign(chosen.data_ptr(), (uint64_t)chosen.size(0), (uint32_t)chosen.size(1), (uint32_t)first, (uint32_t)count,
                                 offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), need ? room.data_ptr() : nullptr, need, on.stream);
        });
        return pack({wrap(offsets), wrap(order), wrap(slots)});
    });
}

// ---- products in 8 bits --------------------------------------------------------
int64_t blocks(int64_t n) { return (n + 127) / 128; }

void eight(const Tensor& q, const char* name) { typed(q, at::ScalarType::Float8_e4m3fn, name, "float8_e4m3fn"); }

// 8-bit numbers: rows at multiples of 16 bytes
void eight_rows(const Tensor& q, const char* name) {
    eight(q, name);
    const int64_t d = q.dim();
    if (q.size(d - 1) > 1 && q.stride(d - 1) != 1) refuse(PyExc_ValueError, "the rows of %s must lie in one piece each", name);
    bool fits = q.numel() == 0 || address(q) % 16 == 0;
    for (int64_t i = 0; i < d - 1; ++i) fits = fits && (q.numel() == 0 || q.size(i) <= 1 || q.stride(i) % 16 == 0);
    if (!fits) refuse(PyExc_ValueError, "the rows of %s must start at multiples of 16 bytes", name);
}
void scales_of(const Tensor& s, at::IntArrayRef size, const Tensor& q, const char* name) {
    same_device(q, s, name);
    typed(s, at::kFloat, name, "float32");
    if (s.sizes() != size) refuse(PyExc_ValueError, "%s must have a number for each block of 128", name);
}
// the distance of neighbours along `dim`, 0 where there are none
int64_t apart(const Tensor& t, int64_t dim) { return t.numel() && t.size(dim) > 1 ? t.stride(dim) : 0; }

// quantise(x): 8-bit numbers and scales by rows
PyObject* host_quantise(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 1);
        const Tensor& x = a.tensor(0, "x");
        rows_of(x, "x");
        const int dtype = code_of(x.scalar_type(), "x");
        const int64_t rows = x.size(0), wide = blocks(x.size(1)) * 128;
        OnDevice on(x.get_device());
        // (scales of a block side by side: products read them for many rows and one block at a time)
        const Tensor q = empty(x, {rows, wide}, at::kByte), scale = empty(x, {wide / 128, rows}, at::kFloat);
        launch("mint_rows8", [&] {
            return native.rows8(x.data_ptr(), x.stride(0), (uint64_t)rows, (uint64_t)x.size(1), dtype, q.data_ptr(), wide, scale.data_ptr(), 1, rows,
                                on.stream);
        });
        return pack({wrap(q.view(at::ScalarType::Float8_e4m3fn).narrow(1, 0, x.size(1))), wrap(scale.t())});
    });
}

// quantise_weight(w): 8-bit numbers and scales by squares, of (rows, depth) or (matrices, rows, depth)
PyObject* host_quantise_weight(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 1);
        const Tensor& w = a.tensor(0, "w");
        const int64_t d = w.dim();
        if (d != 2 && d != 3) refuse(PyExc_ValueError, "w must have 2 or 3 dimensions");
        if (w.size(d - 1) > 1 && w.stride(d - 1) != 1) refuse(PyExc_ValueError, "the rows of w must lie in one piece each");
        const int dtype = code_of(w.scalar_type(), "w");
        const int64_t rows = w.size(d - 2), depth = w.size(d - 1), wide = blocks(depth) * 128, matrices = d == 3 ? w.size(0) : 1;
        OnDevice on(w.get_device());
        const Tensor q = d == 3 ? empty(w, {matrices, rows, wide}, at::kByte) : empty(w, {rows, wide}, at::kByte);
        const Tensor scale = d == 3 ? empty(w, {matrices, blocks(rows), blocks(depth)}, at::kFloat) : empty(w, {blocks(rows), blocks(depth)}, at::kFloat);
        launch("mint_squares8", [&] {
            return native.squares8(w.data_ptr(), d == 3 ? w.stride(0) : 0, w.stride(d - 2), (uint32_t)matrices, (uint64_t)rows, (uint64_t)depth, dtype,
                                   q.data_ptr(), rows * wide, wide, scale.data_ptr(), on.stream);
        });
        return pack({wrap(q.view(at::ScalarType::Float8_e4m3fn).narrow(d - 1, 0, depth)), wrap(scale)});
    });
}

// an assignment's offsets and order
void plan_of(const Tensor& like, const Tensor& offsets, const Tensor& order) {
    same_device(like, offsets, "offsets");
    same_device(like, order, "tokens");
    typed(offsets, at::kInt, "offsets", "int32");
    typed(order, at::kInt, "tokens", "int32");
    dims(offsets, 1, "offsets");
    dims(order, 1, "tokens");
    dense(offsets, "offsets");
    dense(order, "tokens");
    if (offsets.size(0) < 1) refuse(PyExc_ValueError, "offsets must have a number at least");
}
// rows that are gathered by an assignment's tokens, of which its slots, where they are known, have a row each
void gathered(const Args& a, int slots, const Tensor& x) {
    if (a.none(slots)) return;
    const Tensor& t = a.tensor(slots, "slots");
    dims(t, 2, "slots");
    if (x.size(0) < t.size(0)) refuse(PyExc_ValueError, "x has %lld rows, the assignment %lld tokens", (long long)x.size(0), (long long)t.size(0));
}

// product(x, x_scale or None, wq, w_scale, offsets or None, tokens or None, slots or None, gather, dtype, out or None)
PyObject* host_product(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 10);
        const Tensor &x = a.tensor(0, "x"), &w = a.tensor(2, "weight"), &sw = a.tensor(3, "the weight's scale");
        rows_of(x, "x");
        same_device(x, w, "weight");
        const bool by_expert = !a.none(4), gather = a.truth(7);
        if (gather && !by_expert) refuse(PyExc_ValueError, "gather needs an assignment");
        dims(w, by_expert ? 3 : 2, "weight");
        eight_rows(w, "weight");
        const int64_t d = w.dim(), cols = w.size(d - 2), depth = w.size(d - 1);
        if (by_expert) scales_of(sw, {w.size(0), blocks(cols), blocks(depth)}, w, "the weight's scale");
        else scales_of(sw, {blocks(cols), blocks(depth)}, w, "the weight's scale");
        if (x.size(1) != depth) refuse(PyExc_ValueError, "x has rows of %lld, the weight of %lld", (long long)x.size(1), (long long)depth);
        mint_product_op op = {};
        op.kind = MINT_PRODUCT_ROWS;
        int64_t rows = x.size(0);
        if (by_expert) {
            const Tensor &offsets = a.tensor(4, "offsets"), &order = a.tensor(5, "tokens");
            plan_of(x, offsets, order);
            if (offsets.size(0) != w.size(0) + 1) refuse(PyExc_ValueError, "the assignment is to %lld experts, the weight of %lld",
                                                         (long long)offsets.size(0) - 1, (long long)w.size(0));
            if (!gather && order.size(0) != rows) refuse(PyExc_ValueError, "x must have a row for each place of the assignment");
            rows = order.size(0);
            op.experts = (uint32_t)std::min<int64_t>(w.size(0), 0x7FFFFFFF);
            op.offsets = address(offsets);
            op.w_matrix = apart(w, 0);
            op.sw_matrix = apart(sw, 0);
            if (gather) {
                gathered(a, 6, x);
                op.tokens = address(order);
                if (x.size(0) == 0 && rows) refuse(PyExc_ValueError, "x has no rows to gather");
            }
        }
        int64_t code;
        const bool given = !a.none(9);
        if (given) {
            const Tensor& out = a.tensor(9, "out");
            same_device(x, out, "out");
            result(out, rows, cols, "out");
            code = code_of(out.scalar_type(), "out");
            if (!a.none(8) && a.integer(8, "dtype", 0, 2) != code) refuse(PyExc_TypeError, "out is of another type than dtype");
        } else {
            code = a.none(8) ? (int64_t)MINT_BF16 : a.integer(8, "dtype", 0, 2);
        }
        const bool already = !a.none(1);
        if (already) {
            eight_rows(x, "x");
            scales_of(a.tensor(1, "x's scale"), {x.size(0), blocks(depth)}, x, "x's scale");
        } else {
            code_of(x.scalar_type(), "x");
        }
        OnDevice on(x.get_device());
        const Tensor out = given ? a.tensor(9, "out") : empty(x, {rows, cols}, type_of(code));
        op.x = address(x);
        if (already) {
            const Tensor& sx = a.tensor(1, "x's scale");
            op.x_dtype = MINT_BYTES;
            op.x_stride = apart(x, 0);
            op.sx = address(sx);
            op.sx_row = sx.stride(0);
            op.sx_block = sx.stride(1);
        } else {
            op.x_dtype = code_of(x.scalar_type(), "x");
            op.x_stride = x.stride(0);
        }
        op.dtype = (int32_t)code;
        op.w = address(w);
        op.sw = address(sw);
        op.out = address(out);
        op.rows = (uint64_t)rows;
        op.cols = (uint64_t)cols;
        op.depth = (uint64_t)depth;
        op.x_rows = (uint64_t)x.size(0);
        op.w_stride = apart(w, d - 2);
        op.out_stride = rows > 1 ? out.stride(0) : cols;
        op.sw_row = sw.stride(d - 2);
        op.sw_block = sw.stride(d - 1);
        Tensor room;
        if ((op.workspace_bytes = native.product8_workspace(&op))) {
            room = empty(x, {(int64_t)op.workspace_bytes}, at::kByte);
            op.workspace = address(room);
        }
        launch("mint_product8", [&] { return native.product8(&op, on.stream); });
        if (given) return Py_NewRef(list[9]);
        return wrap(out);
    });
}

// weight_grad(d, x, offsets or None, tokens or None, slots or None, gather, dtype)
PyObject* host_weight_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 7);
        const Tensor &d = a.tensor(0, "grad"), &x = a.tensor(1, "x");
        rows_of(d, "grad");
        rows_of(x, "x");
        same_device(x, d, "grad");
        const int d_code = code_of(d.scalar_type(), "grad"), x_code = code_of(x.scalar_type(), "x");
        const bool by_expert = !a.none(2), gather = a.truth(5);
        if (gather && !by_expert) refuse(PyExc_ValueError, "gather needs an assignment");
        mint_weight_grad_op op = {};
        op.d_dtype = d_code;
        op.x_dtype = x_code;
        op.dtype = a.none(6) ? (int32_t)MINT_F32 : (int32_t)a.integer(6, "dtype", 0, 2);
        const int64_t rows = d.size(0), cols = d.size(1), depth = x.size(1);
        int64_t experts = 0;
        if (by_expert) {
            const Tensor &offsets = a.tensor(2, "offsets"), &order = a.tensor(3, "tokens");
            plan_of(x, offsets, order);
            if (order.size(0) != rows) refuse(PyExc_ValueError, "grad must have a row for each place of the assignment");
            experts = offsets.size(0) - 1;
            if (experts > 65535) refuse(PyExc_ValueError, "at most 65535 experts");
            op.offsets = address(offsets);
            if (gather) {
                gathered(a, 4, x);
                op.tokens = address(order);
            }
        }
        if (gather ? x.size(0) == 0 && rows != 0 : x.size(0) != rows) refuse(PyExc_ValueError, "x and grad have different numbers of rows");
        OnDevice on(x.get_device());
        const Tensor out = by_expert ? empty(x, {experts, cols, depth}, type_of(op.dtype)) : empty(x, {cols, depth}, type_of(op.dtype));
        op.d = address(d);
        op.x = address(x);
        op.out = address(out);
        op.rows = (uint64_t)rows;
        op.x_rows = (uint64_t)x.size(0);
        op.cols = (uint64_t)cols;
        op.depth = (uint64_t)depth;
        op.d_stride = d.stride(0);
        op.x_stride = x.stride(0);
        op.out_stride = depth;
        op.out_matrix = cols * depth;
        op.experts = (uint32_t)experts;
        Tensor room;
        if ((op.workspace_bytes = native.weight_grad8_workspace(&op))) {
            room = empty(x, {(int64_t)op.workspace_bytes}, at::kByte);
            op.workspace = address(room);
        }
        launch("mint_weight_grad8", [&] { return native.weight_grad8(&op, on.stream); });
        return wrap(out);
    });
}

// ---- combination -----------------------------------------------------------------
// combine(rows, slots, weights or None, out or None)
PyObject* host_combine(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 4);
        const Tensor &rows = a.tensor(0, "rows"), &slots = a.tensor(1, "slots");
        rows_of(rows, "rows");
        const int dtype = code_of(rows.scalar_type(), "rows");
        same_device(rows, slots, "slots");
        choices(slots, "slots");
        const void* weights = nullptr;
        if (!a.none(2)) {
            const Tensor& w = a.tensor(2, "weights");
            weights_of(w, slots, "weights");
            weights = w.data_ptr();
        }
        const bool given = !a.none(3);
        if (given) {
            const Tensor& out = a.tensor(3, "out");
            same_device(rows, out, "out");
            result(out, slots.size(0), rows.size(1), "out");
            if (out.scalar_type() != rows.scalar_type()) refuse(PyExc_TypeError, "out must be of the rows' type");
        }
        if (rows.size(1) > 0x7FFFFFFF - 8192) refuse(PyExc_ValueError, "the rows are too long");
        OnDevice on(rows.get_device());
        const Tensor out = given ? a.tensor(3, "out") : empty(rows, {slots.size(0), rows.size(1)}, rows.scalar_type());
        launch("mint_combine", [&] {
            return native.combine(rows.data_ptr(), rows.stride(0), (uint64_t)rows.size(0), slots.data_ptr(), weights, (uint64_t)slots.size(0),
                                  (uint32_t)slots.size(1), (uint32_t)rows.size(1), out.data_ptr(), out.stride(0), dtype, on.stream);
        });
        if (given) return Py_NewRef(list[3]);
        return wrap(out);
    });
}

// combine_grad(d_out, rows, offsets, slots, weights or None): (d_rows, d_weights or None)
PyObject* host_combine_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 5);
        const Tensor &d = a.tensor(0, "grad"), &rows = a.tensor(1, "rows"), &offsets = a.tensor(2, "offsets"), &slots = a.tensor(3, "slots");
        rows_of(d, "grad");
        rows_of(rows, "rows");
        const int dtype = code_of(rows.scalar_type(), "rows");
        if (d.scalar_type() != rows.scalar_type()) refuse(PyExc_TypeError, "grad must be of the rows' type");
        same_device(rows, d, "grad");
        same_device(rows, slots, "slots");
        same_device(rows, offsets, "offsets");
        choices(slots, "slots");
        typed(offsets, at::kInt, "offsets", "int32");
        dims(offsets, 1, "offsets");
        dense(offsets, "offsets");
        if (offsets.size(0) < 1) refuse(PyExc_ValueError, "offsets must have a number at least");
        if (d.size(0) != slots.size(0) || d.size(1) != rows.size(1)) refuse(PyExc_ValueError, "grad must be what the combination's result is like");
        if (rows.size(0) != slots.numel()) refuse(PyExc_ValueError, "rows must have one for each place of the assignment");
        if (rows.size(1) > 0x7FFFFFFF - 8192) refuse(PyExc_ValueError, "the rows are too long");
        const void* weights = nullptr;                 // (of no tokens there are none either way)
        const bool weighted = !a.none(4);
        if (weighted) {
            const Tensor& w = a.tensor(4, "weights");
            weights_of(w, slots, "weights");
            weights = w.data_ptr();
        }
        OnDevice on(rows.get_device());
        const Tensor d_rows = empty(rows, rows.sizes(), rows.scalar_type());
        Tensor d_weights;
        if (weighted) d_weights = empty(rows, slots.sizes(), at::kFloat);
        const int32_t* const used = static_cast<const int32_t*>(offsets.data_ptr()) + (offsets.size(0) - 1);
        launch("mint_combine_grad", [&] {
            return native.combine_grad(d.data_ptr(), d.stride(0), rows.data_ptr(), rows.stride(0), (uint64_t)rows.size(0), slots.data_ptr(), weights,
                                       used, (uint64_t)slots.size(0), (uint32_t)slots.size(1), (uint32_t)rows.size(1), d_rows.data_ptr(),
                                       d_rows.stride(0), weighted ? d_weights.data_ptr() : nullptr, dtype, on.stream);
        });
        return pack({wrap(d_rows), weighted ? wrap(d_weights) : Py_NewRef(Py_None)});
    });
}

// ---- norms and the residual stream ------------------------------------------------
// four arguments from `i` on: kind, weight or None, bias or None, eps
void norm_of(const Args& a, int i, const Tensor& like, int64_t width, mint_norm& n, const char* name) {
    n.kind = (int32_t)a.integer(i, "kind", MINT_NORM_NONE, MINT_NORM_LAYER);
    if (n.kind == MINT_NORM_NONE) return;
    n.eps = a.number(i + 3);
    n.dtype = MINT_F32;
    for (int k = 1; k <= 2; ++k) {
        if (a.none(i + k)) continue;
        const Tensor& t = a.tensor(i + k, name);
        same_device(like, t, name);
        dims(t, 1, name);
        dense(t, name);
        if (t.size(0) != width) refuse(PyExc_ValueError, "%s must have a number for each of %lld channels", name, (long long)width);
        const int code = code_of(t.scalar_type(), name);
        if (k == 2 && n.weight && code != n.dtype) refuse(PyExc_TypeError, "%s: weight and bias must be of one type", name);
        n.dtype = code;
        (k == 1 ? n.weight : n.bias) = address(t);
    }
}
// What join and its gradient have in common: stream, y or None, gate or None, gate_by, scale, carry, then after's and before's norm (arguments i .. i + 13)
void join_of(const Args& a, int i, mint_join_op& op) {
    const Tensor& s = a.tensor(i, "stream");
    rows_of(s, "stream");
    op.stream_dtype = code_of(s.scalar_type(), "stream");
    op.dtype = op.stream_dtype;
    op.rows = (uint64_t)s.size(0);
    op.width = (uint64_t)s.size(1);
    if (s.size(0) > 0x7FFFFFFF / 4 || s.size(1) > 0x7FFFFFFF - 8192) refuse(PyExc_ValueError, "stream is too large");
    op.stream = address(s);
    op.stream_stride = s.stride(0);
    op.gate_by = (int32_t)a.integer(i + 3, "gate_by", MINT_ACT_NONE, MINT_ACT_GELU_TANH);
    op.scale = a.number(i + 4);
    op.carry = a.number(i + 5);
    norm_of(a, i + 6, s, s.size(1), op.after, "after");
    norm_of(a, i + 10, s, s.size(1), op.before, "before");
    if (!a.none(i + 1)) {
        const Tensor& y = a.tensor(i + 1, "y");
        same_device(s, y, "y");
        rows_of(y, "y");
        op.dtype = code_of(y.scalar_type(), "y");
        if (op.stream_dtype != op.dtype && op.stream_dtype != MINT_F32) refuse(PyExc_TypeError, "stream must be of y's type or float32");
        if (y.sizes() != s.sizes()) refuse(PyExc_ValueError, "y must be like stream");
        op.y = address(y);
        op.y_stride = y.stride(0);
    }
    if (!a.none(i + 2)) {
        const Tensor& g = a.tensor(i + 2, "gate");
        same_device(s, g, "gate");
        op.gate_dtype = code_of(g.scalar_type(), "gate");
        op.gate = address(g);
        if (g.dim() == 1 && g.size(0) == s.size(1)) {
            dense(g, "gate");
            op.gate_form = MINT_GATE_CHANNEL;
        } else if (g.sizes() == s.sizes()) {
            rows_of(g, "gate");
            op.gate_form = MINT_GATE_ALL;
            op.gate_row = g.stride(0);
        } else if (g.dim() == 2 && g.size(0) == s.size(0) && g.size(1) == 1) {
            op.gate_form = MINT_GATE_ROW;
            op.gate_row = g.stride(0);
        } else {
            refuse(PyExc_ValueError, "gate must be (width,), (rows, 1) or (rows, width)");
        }
    }
}
constexpr int kJoinArguments = 14;

// join(stream, y, gate, gate_by, scale, carry, after x 4, before x 4, dtype or None, out or None): (stream or None, next or None)
PyObject* host_join(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, kJoinArguments + 2);
        mint_join_op op = {};
        join_of(a, 0, op);
        const Tensor& s = a.tensor(0, "stream");
        if (!a.none(kJoinArguments)) {
            const int64_t code = a.integer(kJoinArguments, "dtype", 0, 2);
            if (op.y ? code != op.dtype : code != op.stream_dtype && op.stream_dtype != MINT_F32)
                refuse(PyExc_TypeError, "dtype must be that of y, or of x, or anything if that is float32");
            op.dtype = (int32_t)code;
        }
        const bool block = !a.none(1), next = op.before.kind != MINT_NORM_NONE, given = !a.none(kJoinArguments + 1);
        if (!block && !next) refuse(PyExc_ValueError, "there is neither a block's output nor a norm");
        if (given) {
            const Tensor& out = a.tensor(kJoinArguments + 1, "out");
            same_device(s, out, "out");
            result(out, s.size(0), s.size(1), "out");
            if (code_of(out.scalar_type(), "out") != (block ? op.stream_dtype : op.dtype)) refuse(PyExc_TypeError, "out is of another type than the result");
            clear_of(out, s, block ? "stream" : "x", true);
            if (block) clear_of(out, a.tensor(1, "y"), "y", false);
            for (const auto& [i, name] : {std::pair<int, const char*>{2, "gate"}, {7, "a weight"}, {8, "a bias"}, {11, "a weight"}, {12, "a bias"}})
                if (!a.none(i)) clear_of(out, a.tensor(i, name), name, false);
        }
        OnDevice on(s.get_device());
        Tensor stream, h;
        if (block) {
            stream = given ? a.tensor(kJoinArguments + 1, "out") : empty(s, s.sizes(), s.scalar_type());
            op.new_stream = address(stream);
            op.new_stride = s.size(0) > 1 ? stream.stride(0) : s.size(1);
        }
        if (next) {
            h = given && !block ? a.tensor(kJoinArguments + 1, "out") : empty(s, s.sizes(), type_of(op.dtype));
            op.next = address(h);
            op.next_stride = s.size(0) > 1 ? h.stride(0) : s.size(1);
        }
        launch("mint_join", [&] { return native.join(&op, on.stream); });
        return pack({block ? given ? Py_NewRef(list[kJoinArguments + 1]) : wrap(stream) : Py_NewRef(Py_None),
                     next ? given && !block ? Py_NewRef(list[kJoinArguments + 1]) : wrap(h) : Py_NewRef(Py_None)});
    });
}

// join_grad(d_stream or None, d_next or None, stream, ... as above): (d_stream, d_y, d_gate, d_after_weight, d_after_bias, d_before_weight,
// d_before_bias), None in the place of those that there are none of
PyObject* host_join_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, kJoinArguments + 2);
        mint_join_grad_op op = {};
        join_of(a, 2, op.join);
        const Tensor& s = a.tensor(2, "stream");
        const bool block = !a.none(3);
        if (a.none(0) && a.none(1)) refuse(PyExc_ValueError, "there is no gradient to go on with");
        if (!a.none(1)) {
            const Tensor& d = a.tensor(1, "the norm's grad");
            same_device(s, d, "the norm's grad");
            rows_of(d, "the norm's grad");
            if (d.sizes() != s.sizes()) refuse(PyExc_ValueError, "the norm's grad must be like its result");
            const int code = code_of(d.scalar_type(), "the norm's grad");
            if (block ? code != op.join.dtype : code != op.join.stream_dtype && op.join.stream_dtype != MINT_F32)
                refuse(PyExc_TypeError, "the norm's grad must be of its result's type");
            op.join.dtype = code;
            if (op.join.before.kind == MINT_NORM_NONE) refuse(PyExc_ValueError, "there is no norm that this is the gradient of");
            op.d_next = address(d);
            op.d_next_stride = d.stride(0);
        }
        if (!a.none(0)) {
            const Tensor& d = a.tensor(0, "the stream's grad");
            same_device(s, d, "the stream's grad");
            rows_of(d, "the stream's grad");
            if (d.sizes() != s.sizes()) refuse(PyExc_ValueError, "the stream's grad must be like the stream");
            if (d.scalar_type() != s.scalar_type()) refuse(PyExc_TypeError, "the stream's grad must be of the stream's type");
            op.d_stream = address(d);
            op.d_stream_stride = d.stride(0);
        }
        OnDevice on(s.get_device());
        const auto make = [&](int i, uint64_t& at) {
            if (a.none(i)) return Tensor();
            const Tensor& like = a.tensor(i, "a weight");
            Tensor t = empty(like, like.sizes(), like.scalar_type());
            at = address(t);
            return t;
        };
        const Tensor to_stream = empty(s, s.sizes(), s.scalar_type());
        op.to_stream = address(to_stream);
        op.to_stream_stride = s.size(1);
        Tensor to_y, to_gate, aw, ab, bw, bb;
        if (block) {
            to_y = empty(s, s.sizes(), type_of(op.join.dtype));
            op.to_y = address(to_y);
            op.to_y_stride = s.size(1);
            to_gate = make(4, op.to_gate);
            op.to_gate_stride = op.join.gate_form == MINT_GATE_ALL ? s.size(1) : 1;
            if (op.join.after.kind) {
                aw = make(9, op.to_after_weight);
                ab = make(10, op.to_after_bias);
            }
        }
        if (op.join.before.kind) {
            bw = make(13, op.to_before_weight);
            bb = make(14, op.to_before_bias);
        }
        Tensor room;
        if ((op.workspace_bytes = native.join_grad_workspace(&op))) {
            room = empty(s, {(int64_t)op.workspace_bytes}, at::kByte);
            op.workspace = address(room);
        }
        launch("mint_join_grad", [&] { return native.join_grad(&op, on.stream); });
        const auto give = [](const Tensor& t) { return t.defined() ? wrap(t) : Py_NewRef(Py_None); };
        return pack({wrap(to_stream), give(to_y), give(to_gate), give(aw), give(ab), give(bw), give(bb)});
    });
}

// ---- dense products ------------------------------------------------------------------
void dense_launch(mint_dense_op& op, const Tensor& like, OnDevice& on) {
    Tensor room;
    if ((op.workspace_bytes = native.dense_workspace(&op))) {
        room = empty(like, {(int64_t)op.workspace_bytes}, at::kByte);
        op.workspace = address(room);
    }
    launch("mint_dense", [&] { return native.dense(&op, on.stream); });
}
// both operands of a dense product
void operands(const Tensor& x, const Tensor& w, const char* x_name, const char* w_name, mint_dense_op& op) {
    rows_of(x, x_name);
    rows_of(w, w_name);
    same_device(x, w, w_name);
    op.dtype = code_of(x.scalar_type(), x_name);
    if (w.scalar_type() != x.scalar_type()) refuse(PyExc_TypeError, "%s must be of the type of %s", w_name, x_name);
    op.x = address(x);
    op.w = address(w);
    op.x_stride = x.stride(0);
    op.w_stride = w.stride(0);
}
// the result's type, where one is named or `out` is given, and the result
Tensor dense_out(const Args& a, int dtype_at, int out_at, const Tensor& x, int64_t rows, int64_t cols, mint_dense_op& op) {
    int64_t code = a.none(dtype_at) ? op.dtype : a.integer(dtype_at, "dtype", 0, 2);
    const bool given = out_at >= 0 && !a.none(out_at);
    if (given) {
        const Tensor& out = a.tensor(out_at, "out");
        same_device(x, out, "out");
        result(out, rows, cols, "out");
        const int of_out = code_of(out.scalar_type(), "out");
        if (!a.none(dtype_at) && code != of_out) refuse(PyExc_TypeError, "out is of another type than dtype");
        code = of_out;
    }
    if (code != op.dtype && code != MINT_F32) refuse(PyExc_TypeError, "the result must be of the operands' type or float32");
    op.out_dtype = (int32_t)code;
    const Tensor out = given ? a.tensor(out_at, "out") : empty(x, {rows, cols}, type_of(code));
    op.out = address(out);
    op.out_stride = rows > 1 ? out.stride(0) : cols;
    op.rows = (uint64_t)rows;
    op.cols = (uint64_t)cols;
    return out;
}

// dense_product(x, weight, bias or None, activation, residual or None, keep, dtype or None, out or None): out, or (out, z)
PyObject* host_dense_product(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 8);
        const Tensor &x = a.tensor(0, "x"), &w = a.tensor(1, "weight");
        mint_dense_op op = {};
        op.form = MINT_DENSE_PRODUCT;
        operands(x, w, "x", "weight", op);
        if (x.size(1) != w.size(1)) refuse(PyExc_ValueError, "x has rows of %lld, the weight of %lld", (long long)x.size(1), (long long)w.size(1));
        const int64_t rows = x.size(0), cols = w.size(0);
        op.depth = (uint64_t)x.size(1);
        if (!a.none(2)) {
            const Tensor& b = a.tensor(2, "bias");
            same_device(x, b, "bias");
            dims(b, 1, "bias");
            dense(b, "bias");
            if (b.scalar_type() != x.scalar_type()) refuse(PyExc_TypeError, "bias must be of x's type");
            if (b.size(0) != cols) refuse(PyExc_ValueError, "bias must have a number for each of %lld columns", (long long)cols);
            op.bias = address(b);
        }
        op.activation = (int32_t)a.integer(3, "activation", MINT_ACT_NONE, MINT_ACT_GELU_TANH);
        const bool keep = a.truth(5), given = !a.none(7);
        OnDevice on(x.get_device());
        const Tensor out = dense_out(a, 6, 7, x, rows, cols, op);
        if (!a.none(4)) {
            const Tensor& r = a.tensor(4, "residual");
            same_device(x, r, "residual");
            rows_of(r, "residual");
            if (r.size(0) != rows || r.size(1) != cols) refuse(PyExc_ValueError, "residual must be (%lld, %lld)", (long long)rows, (long long)cols);
            if (code_of(r.scalar_type(), "residual") != op.out_dtype) refuse(PyExc_TypeError, "residual must be of the result's type");
            op.residual = address(r);
            op.residual_stride = r.stride(0);
        }
        if (given) {
            clear_of(out, x, "x", false);
            clear_of(out, w, "the weight", false);
            if (!a.none(2)) clear_of(out, a.tensor(2, "bias"), "bias", false);
            if (!a.none(4)) clear_of(out, a.tensor(4, "residual"), "residual", true);
        }
        Tensor z;
        if (keep) {
            z = empty(x, {rows, cols}, x.scalar_type());
            op.z = address(z);
            op.z_stride = cols;
        }
        dense_launch(op, x, on);
        PyObject* const result = given ? Py_NewRef(list[7]) : wrap(out);
        return keep ? pack({result, wrap(z)}) : result;
    });
}
// dense_input_grad(grad, weight, dtype or None)
PyObject* host_dense_input_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 3);
        const Tensor &d = a.tensor(0, "grad"), &w = a.tensor(1, "weight");
        mint_dense_op op = {};
        op.form = MINT_DENSE_INPUT_GRAD;
        operands(d, w, "grad", "weight", op);
        if (d.size(1) != w.size(0)) refuse(PyExc_ValueError, "grad has rows of %lld, the weight %lld rows", (long long)d.size(1), (long long)w.size(0));
        op.depth = (uint64_t)w.size(0);
        OnDevice on(d.get_device());
        const Tensor out = dense_out(a, 2, -1, d, d.size(0), w.size(1), op);
        dense_launch(op, d, on);
        return wrap(out);
    });
}
// dense_weight_grad(grad, x, dtype or None)
PyObject* host_dense_weight_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 3);
        const Tensor &d = a.tensor(0, "grad"), &x = a.tensor(1, "x");
        mint_dense_op op = {};
        op.form = MINT_DENSE_WEIGHT_GRAD;
        operands(d, x, "grad", "x", op);
        if (d.size(0) != x.size(0)) refuse(PyExc_ValueError, "x and grad have different numbers of rows");
        op.depth = (uint64_t)x.size(0);
        OnDevice on(d.get_device());
        const Tensor out = dense_out(a, 2, -1, d, d.size(1), x.size(1), op);
        dense_launch(op, d, on);
        return wrap(out);
    });
}
// activation_grad(grad, z or None, activation, bias, dtype): (d_z, d_bias or None)
PyObject* host_activation_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 5);
        const Tensor& d = a.tensor(0, "grad");
        rows_of(d, "grad");
        mint_activation_grad_op op = {};
        op.d_dtype = code_of(d.scalar_type(), "grad");
        op.activation = (int32_t)a.integer(2, "activation", MINT_ACT_NONE, MINT_ACT_GELU_TANH);
        const bool bias = a.truth(3);
        if (!a.none(1)) {
            const Tensor& z = a.tensor(1, "z");
            same_device(d, z, "z");
            rows_of(z, "z");
            if (z.sizes() != d.sizes()) refuse(PyExc_ValueError, "z must be like grad");
            op.dtype = code_of(z.scalar_type(), "z");
            if (!a.none(4) && a.integer(4, "dtype", 0, 2) != op.dtype) refuse(PyExc_TypeError, "z is of another type than dtype");
            op.z = address(z);
            op.z_stride = z.stride(0);
        } else {
            if (op.activation != MINT_ACT_NONE) refuse(PyExc_ValueError, "z is wanted: what the activation was applied to");
            op.dtype = a.none(4) ? op.d_dtype : (int32_t)a.integer(4, "dtype", 0, 2);
        }
        if (op.d_dtype != op.dtype && op.d_dtype != MINT_F32) refuse(PyExc_TypeError, "grad must be of the operands' type or float32");
        op.rows = (uint64_t)d.size(0);
        op.cols = (uint64_t)d.size(1);
        op.d = address(d);
        op.d_stride = d.stride(0);
        // (without an activation there may be nothing to change)
        const bool same = op.activation == MINT_ACT_NONE && op.dtype == op.d_dtype;
        OnDevice on(d.get_device());
        Tensor d_z, d_bias, room;
        if (!same) {
            d_z = empty(d, d.sizes(), type_of(op.dtype));
            op.d_z = address(d_z);
            op.d_z_stride = d.size(1);
        }
        if (bias) {
            d_bias = empty(d, {d.size(1)}, type_of(op.dtype));
            op.d_bias = address(d_bias);
            if ((op.workspace_bytes = native.activation_grad_workspace(op.rows, op.cols))) {
                room = empty(d, {(int64_t)op.workspace_bytes}, at::kByte);
                op.workspace = address(room);
            }
        }
        launch("mint_activation_grad", [&] { return native.activation_grad(&op, on.stream); });
        return pack({same ? Py_NewRef(list[0]) : wrap(d_z), bias ? wrap(d_bias) : Py_NewRef(Py_None)});
    });
}

// ---- the loss that balances experts ----------------------------------------------------
// logits, experts, score, offsets or None, z: arguments i .. i + 4
void balance_of(const Args& a, int i, mint_balance_op& op) {
    const Tensor &x = a.tensor(i, "logits"), &chosen = a.tensor(i + 1, "experts");
    rows_of(x, "logits");
    same_device(x, chosen, "experts");
    choices(chosen, "experts");
    if (x.size(1) < 1 || x.size(1) > 1024) refuse(PyExc_ValueError, "logits must be of 1..1024 experts");
    if (chosen.size(0) != x.size(0) || chosen.size(1) > 1024) refuse(PyExc_ValueError, "experts must be what was chosen by these logits");
    op.dtype = code_of(x.scalar_type(), "logits");
    op.logits = address(x);
    op.chosen = address(chosen);
    op.row_stride = x.stride(0);
    op.tokens = (uint64_t)x.size(0);
    op.experts = (uint32_t)x.size(1);
    op.topk = (uint32_t)chosen.size(1);
    op.score = (int32_t)a.integer(i + 2, "score", 0, 1);
    op.sequences = 1;
    if (!a.none(i + 3)) {
        const Tensor& offsets = a.tensor(i + 3, "offsets");
        same_device(x, offsets, "offsets");
        typed(offsets, at::kInt, "offsets", "int32");
        dims(offsets, 1, "offsets");
        dense(offsets, "offsets");
        if (offsets.size(0) < 2) refuse(PyExc_ValueError, "offsets must have two numbers at least");
        if (offsets.size(0) - 1 > 0xFFFF) refuse(PyExc_ValueError, "at most %d sequences", 0xFFFF);
        op.offsets = address(offsets);
        op.sequences = (uint64_t)offsets.size(0) - 1;
    }
    op.z = a.number(i + 4);
}
// balance(logits, experts, score, offsets or None, z): (loss, counts, shares, there)
PyObject* host_balance(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 5);
        mint_balance_op op = {};
        balance_of(a, 0, op);
        const Tensor& x = a.tensor(0, "logits");
        const int64_t s = (int64_t)op.sequences, e = op.experts;
        OnDevice on(x.get_device());
        const Tensor loss = empty(x, {}, at::kFloat), counts = empty(x, {s, e}, at::kInt), shares = empty(x, {s, e}, at::kFloat),
                     there = empty(x, {s}, at::kInt);
        const size_t need = native.balance_workspace(&op);
        Tensor room;
        if (need) room = empty(x, {(int64_t)need}, at::kByte);
        launch("mint_balance", [&] {
            return native.balance(&op, address(loss), address(counts), address(shares), address(there), need ? room.data_ptr() : nullptr, need, on.stream);
        });
        return pack({wrap(loss), wrap(counts), wrap(shares), wrap(there)});
    });
}
// balance_grad(grad, logits, experts, score, offsets or None, z, counts, there, add or None)
PyObject* host_balance_grad(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Args a(list, n, 9);
        mint_balance_op op = {};
        balance_of(a, 1, op);
        const Tensor &d = a.tensor(0, "grad"), &x = a.tensor(1, "logits"), &counts = a.tensor(6, "counts"), &there = a.tensor(7, "there");
        same_device(x, d, "grad");
        same_device(x, counts, "counts");
        same_device(x, there, "there");
        typed(d, at::kFloat, "grad", "float32");
        typed(counts, at::kInt, "counts", "int32");
        typed(there, at::kInt, "there", "int32");
        dense(counts, "counts");
        dense(there, "there");
        if (d.numel() != 1) refuse(PyExc_ValueError, "grad must be one number");
        if (counts.dim() != 2 || counts.size(0) != (int64_t)op.sequences || counts.size(1) != (int64_t)op.experts || there.dim() != 1 ||
            there.size(0) != (int64_t)op.sequences)
            refuse(PyExc_ValueError, "counts and there must be of these sequences and experts");
        uint64_t add = 0;
        int64_t add_stride = 0;
        if (!a.none(8)) {
            const Tensor& more = a.tensor(8, "add");
            same_device(x, more, "add");
            rows_of(more, "add");
            if (more.sizes() != x.sizes()) refuse(PyExc_ValueError, "add must be like logits");
            if (more.scalar_type() != x.scalar_type()) refuse(PyExc_TypeError, "add must be of the logits' type");
            add = address(more);
            add_stride = more.stride(0);
        }
        OnDevice on(x.get_device());
        const Tensor out = empty(x, x.sizes(), x.scalar_type());
        launch("mint_balance_grad", [&] {
            return native.balance_grad(&op, address(d), address(counts), address(there), add, add_stride, address(out), x.size(1), on.stream);
        });
        return wrap(out);
    });
}

// bind(check, addresses in the order of Native's)
PyObject* host_bind(PyObject*, PyObject* const* list, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        constexpr int count = offsetof(Native, check) / sizeof(void*);
        const Args a(list, n, 1 + count);
        void* p[count];
        for (int i = 0; i < count; ++i) {
            p[i] = PyLong_AsVoidPtr(list[1 + i]);
            if (!p[i] && PyErr_Occurred()) throw Raised();
        }
        memcpy(&native, p, sizeof(p));
        Py_INCREF(list[0]);
        Py_XSETREF(native.check, list[0]);
        Py_RETURN_NONE;
    });
}

#define MINT_METHOD(name) {#name, (PyCFunction)(void (*)(void))host_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MINT_METHOD(bind), MINT_METHOD(route), MINT_METHOD(route_grad), MINT_METHOD(assign), MINT_METHOD(quantise),
                         MINT_METHOD(quantise_weight), MINT_METHOD(product), MINT_METHOD(weight_grad), MINT_METHOD(combine),
                         MINT_METHOD(combine_grad), MINT_METHOD(join), MINT_METHOD(join_grad), MINT_METHOD(dense_product),
                         MINT_METHOD(dense_input_grad), MINT_METHOD(dense_weight_grad), MINT_METHOD(activation_grad), MINT_METHOD(balance),
                         MINT_METHOD(balance_grad), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_expert_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__expert_host(void) {
    PyObject* m = PyModule_Create(&module);
    if (!m) return nullptr;
    const size_t bytes[] = {sizeof(mint_route_op), sizeof(mint_product_op), sizeof(mint_weight_grad_op), sizeof(mint_join_op),
                            sizeof(mint_join_grad_op), sizeof(mint_dense_op), sizeof(mint_activation_grad_op), sizeof(mint_balance_op)};
    constexpr Py_ssize_t kinds = sizeof(bytes) / sizeof(bytes[0]);
    PyObject* const list = PyTuple_New(kinds);
    for (Py_ssize_t i = 0; list && i < kinds; ++i) PyTuple_SET_ITEM(list, i, PyLong_FromSize_t(bytes[i]));
    if (!list || PyModule_AddObject(m, "DESCRIPTOR_BYTES", list) < 0) {
        Py_XDECREF(list);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
