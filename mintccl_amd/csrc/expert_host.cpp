// mintccl_amd._expert_host: the host side of the expert layer's operators (routing.py, block8.py,
// combine.py), native: a call for one token takes the GPU a few us, and so must the checks of
// its arguments, its outputs' allocation and the launch.  What a call allocates for itself
// comes from torch's allocator on the calling thread's current stream, on which it launches too.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
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
        // (a result without a history would end the gradient here without a word)
        if (history && t.requires_grad() && c10::GradMode::is_enabled())
            refuse(PyExc_RuntimeError, "%s requires a gradient, and these operators record none: detach it, or call under torch.no_grad()", name);
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
                         MINT_METHOD(combine_grad), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_expert_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__expert_host(void) {
    PyObject* m = PyModule_Create(&module);
    if (!m) return nullptr;
    PyModule_AddIntConstant(m, "ROUTE_BYTES", sizeof(mint_route_op));
    PyModule_AddIntConstant(m, "PRODUCT_BYTES", sizeof(mint_product_op));
    PyModule_AddIntConstant(m, "WEIGHT_GRAD_BYTES", sizeof(mint_weight_grad_op));
    return m;
}
