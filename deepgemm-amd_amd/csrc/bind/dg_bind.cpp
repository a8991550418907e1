// Native half of the Python binding: the calls of a model's step, whose GPU time is
// of the order of the interpreter's at decode sizes, go from torch tensors to the C ABI
// here, without ctypes structures in between. Every check of the
// arguments' values stays in the library; this file only describes tensors
// (dg_tensor) and passes the status back.
//
// Host time of a call, through ctypes -> here (us): 64 x 2112 x 7168 with its workspace
// (two launches) 22.7 -> 9.6, 1 x 256 x 512 16.0 -> 4.9, the cast of 8 x 512 with its
// two allocations 15.1 -> 7.9.
//
// The entry points' addresses come from the ctypes-loaded library (init), so both
// bindings use the same one, whichever that is.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "deepgemm_mi355x.h"

namespace {

struct EntryPoints {
    decltype(&dg_fp8_fp4_gemm_nt) gemm_nt;
    decltype(&dg_fp8_fp4_gemm_nt_ws) gemm_nt_ws;
    decltype(&dg_fp8_gemm_nt_workspace_size) workspace_size;
    decltype(&dg_m_grouped_fp8_fp4_gemm_nt_contiguous) contiguous;
    decltype(&dg_m_grouped_fp8_fp4_gemm_nt_masked) masked;
    decltype(&dg_per_token_cast_to_fp8) cast;
    decltype(&dg_moe_dispatch) dispatch;
    decltype(&dg_moe_swiglu_apply_weight_to_fp8) swiglu;
    decltype(&dg_m_grouped_fp8_gemm_nt_contiguous_swiglu) contiguous_swiglu;
    decltype(&dg_m_grouped_fp8_gemm_nt_masked_swiglu) masked_swiglu;
    decltype(&dg_moe_combine) combine;
    decltype(&dg_m_grouped_bf16_gemm_nt_ragged) ragged_nt;
    decltype(&dg_m_grouped_bf16_gemm_nn_ragged) ragged_nn;
    decltype(&dg_k_grouped_bf16_gemm_tn_ragged) ragged_tn;
    decltype(&dg_bf16_gemm_ragged_workspace_size) ragged_workspace_size;
    decltype(&dg_moe_swiglu_checkpoint) swiglu_checkpoint;
    decltype(&dg_moe_swiglu_backward) swiglu_backward;
} g_entry{};

struct TypeMismatch : std::runtime_error {
    using std::runtime_error::runtime_error;
};

// DG_* code of a tensor's type, or -1 (as the ctypes binding's table).
int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return DG_F32;
        case at::kBFloat16: return DG_BF16;
        case at::kFloat8_e4m3fn: return DG_E4M3;
        case at::kInt: return DG_I32;
        case at::kChar: return DG_I8;
        case at::kByte: return DG_U8;
        case at::kHalf: return DG_F16;
        case at::kLong: return DG_I64;
        case at::ScalarType::Float4_e2m1fn_x2: return DG_I8;
        default: return -1;
    }
}

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) throw TypeMismatch(std::string("expected a torch.Tensor, got ") + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

// A described argument: the struct, and NULL for None where the ABI takes NULL.
struct Arg {
    dg_tensor d{};
    bool given = true;

    void fill(const at::Tensor& t) {
        const int code = dtype_code(t.scalar_type());
        if (code < 0)
            throw std::runtime_error(std::string("Assertion error (_ffi.py): unsupported dtype ") +
                                     c10::toString(t.scalar_type()));
        const auto sizes = t.sizes();
        const auto strides = t.strides();
        if (sizes.size() > 4)
            throw std::runtime_error("Assertion error (_ffi.py): tensors of rank > 4 are not supported");
        d.data = t.data_ptr();
        d.dtype = code;
        d.ndim = (int32_t)sizes.size();
        for (size_t i = 0; i < sizes.size(); ++i) {
            d.sizes[i] = sizes[i];
            d.strides[i] = strides[i];
        }
        d.device = t.is_cuda() ? (int32_t)t.get_device() : -1;
    }
    Arg() : given(false) {}
    explicit Arg(PyObject* o, bool optional = false) {
        if (optional && o == Py_None) given = false;
        else fill(tensor(o));
    }
    const dg_tensor* get() const { return given ? &d : nullptr; }
};

// Integers (the ABI's are 32 bits wide: a longer one is refused, not cut); a pointer argument
// (a ctypes structure's address) is 0 for NULL.
int32_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw TypeMismatch("");
    if (v != (int32_t)v) {
        PyErr_Format(PyExc_OverflowError, "%lld does not fit a 32-bit integer", v);
        throw TypeMismatch("");
    }
    return (int32_t)v;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw TypeMismatch("");
    return (float)v;
}
template <typename T>
T* pointer(PyObject* o) {
    void* p = PyLong_AsVoidPtr(o);
    if (p == nullptr && PyErr_Occurred()) throw TypeMismatch("");
    return static_cast<T*>(p);
}

// Runs f without the GIL: a launch blocks while the stream's queue is full (or its module
// loads), an allocation while the device synchronizes, and the other threads run
// meanwhile, as through ctypes. f sees plain values and C++ tensors only.
template <typename F>
auto unlocked(F&& f) {
    struct Released {
        PyThreadState* state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
    } released;
    return f();
}
template <typename E, typename... A>
int32_t call(E entry, A... args) {
    return unlocked([&] { return entry(args...); });
}

// Runs f with exceptions turned into Python's: nothing leaves these functions.
template <typename F>
PyObject* guarded(Py_ssize_t nargs, Py_ssize_t want, F&& f) {
    if (nargs != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, nargs);
        return nullptr;
    }
    try {
        return PyLong_FromLong(f());
    } catch (const TypeMismatch& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, e.what());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// init(addresses of the entry points up to combine, in EntryPoints' order)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        auto set = [&](auto& entry, int i) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(pointer<void>(a[i])); };
        set(g_entry.gemm_nt, 0), set(g_entry.gemm_nt_ws, 1), set(g_entry.workspace_size, 2);
        set(g_entry.contiguous, 3), set(g_entry.masked, 4), set(g_entry.cast, 5), set(g_entry.dispatch, 6);
        set(g_entry.swiglu, 7), set(g_entry.contiguous_swiglu, 8), set(g_entry.masked_swiglu, 9);
        set(g_entry.combine, 10);
        return 0;
    });
}

// init_bf16(addresses of the entry points after combine)
PyObject* init_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&] {
        auto set = [&](auto& entry, int i) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(pointer<void>(a[i])); };
        set(g_entry.ragged_nt, 0), set(g_entry.ragged_nn, 1), set(g_entry.ragged_tn, 2);
        set(g_entry.ragged_workspace_size, 3);
        set(g_entry.swiglu_checkpoint, 4), set(g_entry.swiglu_backward, 5);
        return 0;
    });
}

// gemm_nt(a, sfa, b, sfb, d, c | None, recipe, disable_ue8m0_cast, epilogue, stream)
PyObject* gemm_nt(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        const Arg ta(a[0]), sfa(a[1]), tb(a[2]), sfb(a[3]), d(a[4]), c(a[5], true);
        const auto* recipe = pointer<const dg_recipe>(a[6]);
        const int32_t disable = integer(a[7]);
        const auto* epilogue = pointer<const dg_epilogue>(a[8]);
        void* stream = pointer<void>(a[9]);
        // Decode-sized calls (at most 64 rows) split K over workgroups when given a
        // workspace: it comes from torch's caching allocator on the output's device
        // and current stream, and goes back to it once the launches are queued.
        if (!c.given && ta.d.ndim == 2 && tb.d.ndim > 0 && ta.d.sizes[0] <= 64 && d.d.dtype == DG_BF16) {
            const int64_t bytes = g_entry.workspace_size(ta.d.sizes[0], tb.d.sizes[0], ta.d.sizes[1]);
            if (bytes > 0) {
                const auto options = tensor(a[4]).options().dtype(at::kByte);
                const at::Tensor ws = unlocked([&] { return at::empty({bytes}, options); });
                Arg w;
                w.fill(ws);
                return call(g_entry.gemm_nt_ws, ta.get(), sfa.get(), tb.get(), sfb.get(), d.get(), nullptr, recipe,
                            disable, epilogue, &w.d, stream);
            }
        }
        return call(g_entry.gemm_nt, ta.get(), sfa.get(), tb.get(), sfb.get(), d.get(), c.get(), recipe, disable,
                    epilogue, stream);
    });
}

// contiguous(a, sfa, b, sfb, d, layout, recipe, disable, psum, zero_padding, expected_m, epilogue, stream)
PyObject* contiguous(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&] {
        const Arg ta(a[0]), sfa(a[1]), tb(a[2]), sfb(a[3]), d(a[4]), layout(a[5]);
        return call(g_entry.contiguous, ta.get(), sfa.get(), tb.get(), sfb.get(), d.get(), layout.get(),
                    pointer<const dg_recipe>(a[6]), integer(a[7]), integer(a[8]),
                    integer(a[9]), integer(a[10]), pointer<const dg_epilogue>(a[11]),
                    pointer<void>(a[12]));
    });
}

// masked(a, sfa, b, sfb, d, masked_m, expected_m, recipe, disable, epilogue, stream)
PyObject* masked(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const Arg ta(a[0]), sfa(a[1]), tb(a[2]), sfb(a[3]), d(a[4]), masked_m(a[5]);
        return call(g_entry.masked, ta.get(), sfa.get(), tb.get(), sfb.get(), d.get(), masked_m.get(),
                    integer(a[6]), pointer<const dg_recipe>(a[7]), integer(a[8]),
                    pointer<const dg_epilogue>(a[9]), pointer<void>(a[10]));
    });
}

// cast(x, q, sf, gran_k, use_ue8m0, stream)
PyObject* cast(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&] {
        const Arg x(a[0]), q(a[1]), sf(a[2]);
        return call(g_entry.cast, x.get(), q.get(), sf.get(), integer(a[3]), integer(a[4]),
                    pointer<void>(a[5]));
    });
}

// dispatch(x, x_sf, topk, topk_weights | None, experts, layout, alignment, a, sf, grouped_layout, pos,
//          row_weights | None, workspace, stream)
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&] {
        const Arg x(a[0]), x_sf(a[1]), topk(a[2]), topk_w(a[3], true), out(a[7]), sf(a[8]), layout(a[9]), pos(a[10]),
            w(a[11], true), ws(a[12]);
        return call(g_entry.dispatch, x.get(), x_sf.get(), topk.get(), topk_w.get(), integer(a[4]),
                    integer(a[5]), integer(a[6]), out.get(), sf.get(), layout.get(), pos.get(),
                    w.get(), ws.get(), pointer<void>(a[13]));
    });
}

// swiglu(x, row_weights | None, row_layout | None, clamp, q, sf, gran_k, stream)
PyObject* swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Arg x(a[0]), w(a[1], true), layout(a[2], true), q(a[4]), sf(a[5]);
        return call(g_entry.swiglu, x.get(), w.get(), layout.get(), real(a[3]), q.get(), sf.get(),
                    integer(a[6]), pointer<void>(a[7]));
    });
}

// contiguous_swiglu(a, sfa, b, sfb, layout, row_weights | None, clamp, q, sf, psum, zero_padding, stream)
PyObject* contiguous_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const Arg ta(a[0]), sfa(a[1]), tb(a[2]), sfb(a[3]), layout(a[4]), w(a[5], true), q(a[7]), sf(a[8]);
        return call(g_entry.contiguous_swiglu, ta.get(), sfa.get(), tb.get(), sfb.get(), layout.get(), w.get(),
                    real(a[6]), q.get(), sf.get(), integer(a[9]), integer(a[10]),
                    pointer<void>(a[11]));
    });
}

// masked_swiglu(a, sfa, b, sfb, masked_m, expected_m, row_weights | None, clamp, q, sf, stream)
PyObject* masked_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const Arg ta(a[0]), sfa(a[1]), tb(a[2]), sfb(a[3]), masked_m(a[4]), w(a[6], true), q(a[8]), sf(a[9]);
        return call(g_entry.masked_swiglu, ta.get(), sfa.get(), tb.get(), sfb.get(), masked_m.get(),
                    integer(a[5]), w.get(), real(a[7]), q.get(), sf.get(), pointer<void>(a[10]));
    });
}

// combine(y, pos, topk_weights | None, out, stream)
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const Arg y(a[0]), pos(a[1]), w(a[2], true), out(a[3]);
        return call(g_entry.combine, y.get(), pos.get(), w.get(), out.get(), pointer<void>(a[4]));
    });
}

// The workspace of a ragged product, from torch's caching allocator on the output's device
// and current stream (it goes back there once the launches are queued); undefined if none.
struct Workspace {
    at::Tensor tensor;
    Arg arg;
    Workspace(int form, const at::Tensor& out, int64_t rows, int64_t m, int64_t n, int64_t k, int64_t groups) {
        const int64_t bytes = out.is_cuda() ? g_entry.ragged_workspace_size(form, rows, m, n, k, (int32_t)groups) : 0;
        if (bytes <= 0) return;   // (-1: sizes that the call itself refuses)
        tensor = unlocked([&] { return at::empty({bytes}, out.options().dtype(at::kByte)); });
        arg.fill(tensor);
        arg.given = true;
    }
};

// m_grouped_ragged(nn, a, b, d, group_ends, alignment, stream)
PyObject* m_grouped_ragged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&] {
        const bool nn = integer(a[0]) != 0;
        const auto entry = nn ? g_entry.ragged_nn : g_entry.ragged_nt;
        const Arg ta(a[1]), tb(a[2]), d(a[3]), ends(a[4]);
        const int32_t alignment = integer(a[5]);
        void* stream = pointer<void>(a[6]);
        const bool fits = ta.d.ndim == 2 && tb.d.ndim == 3;
        const Workspace ws(nn, tensor(a[3]), fits ? ta.d.sizes[0] : 0, 0, tb.d.sizes[nn ? 2 : 1], ta.d.sizes[1], tb.d.sizes[0]);
        return call(entry, ta.get(), tb.get(), d.get(), ends.get(), alignment, ws.arg.get(), stream);
    });
}

// k_grouped_ragged(a, b, b_sf | None, d, group_ends, c | None, alignment, stream)
PyObject* k_grouped_ragged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Arg ta(a[0]), tb(a[1]), sf(a[2], true), d(a[3]), ends(a[4]), c(a[5], true);
        const int32_t alignment = integer(a[6]);
        void* stream = pointer<void>(a[7]);
        const bool fits = ta.d.ndim == 2 && tb.d.ndim == 2 && d.d.ndim == 3;
        const Workspace ws(sf.given ? 3 : 2, tensor(a[3]), ta.d.sizes[0], ta.d.sizes[1], fits ? tb.d.sizes[1] : 0, 0, d.d.sizes[0]);
        return call(g_entry.ragged_tn, ta.get(), tb.get(), sf.get(), d.get(), ends.get(), c.get(), alignment, ws.arg.get(),
                    stream);
    });
}

// Like guarded, for functions that return the status and new tensors: f() gives both.
template <typename F>
PyObject* guarded_new(Py_ssize_t nargs, Py_ssize_t want, F&& f) {
    int32_t status = 0;
    std::vector<at::Tensor> out;
    PyObject* done = guarded(nargs, want, [&] {
        std::tie(status, out) = f();
        return status;
    });
    if (done == nullptr) return nullptr;
    PyObject* tuple = PyTuple_New((Py_ssize_t)out.size() + 1);
    if (tuple == nullptr) {
        Py_DECREF(done);
        return nullptr;
    }
    PyTuple_SET_ITEM(tuple, 0, done);
    for (size_t i = 0; i < out.size(); ++i) {
        PyObject* t = out[i].defined() ? THPVariable_Wrap(out[i]) : Py_NewRef(Py_None);
        if (t == nullptr) {
            Py_DECREF(tuple);
            return nullptr;
        }
        PyTuple_SET_ITEM(tuple, (Py_ssize_t)i + 1, t);
    }
    return tuple;
}
using NewTensors = std::pair<int32_t, std::vector<at::Tensor>>;

at::Tensor new_matrix(const at::Tensor& like, int64_t rows, int64_t cols, at::ScalarType type) {
    return at::empty({rows, cols}, like.options().dtype(type));
}

// swiglu_checkpoint(x, row_weights | None, row_layout | None, clamp, stream) -> (status, h, q, sf)
// (the three allocations here, not in Python: 33 x 1024 11.5 -> 9.0 us a call)
PyObject* swiglu_checkpoint(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 5, [&]() -> NewTensors {
        const Arg x(a[0]), w(a[1], true), layout(a[2], true);
        const float clamp = real(a[3]);
        void* stream = pointer<void>(a[4]);
        const at::Tensor& like = tensor(a[0]);
        const bool matrix = x.d.ndim == 2;   // (otherwise the call refuses x)
        const int64_t m = matrix ? x.d.sizes[0] : 0, i = matrix ? x.d.sizes[1] / 2 : 0;
        at::Tensor h, q, sf;
        unlocked([&] {
            h = new_matrix(like, m, i, at::kBFloat16);
            q = new_matrix(like, m, 2 * i, at::kFloat8_e4m3fn);
            sf = new_matrix(like, m, 2 * ((i + 127) / 128), at::kFloat);
            return 0;
        });
        Arg dh, dq, ds;
        dh.fill(h), dq.fill(q), ds.fill(sf);
        return {call(g_entry.swiglu_checkpoint, x.get(), w.get(), layout.get(), clamp, &dh.d, &dq.d, &ds.d, stream),
                {h, q, sf}};
    });
}

// swiglu_backward(dh, q, sf, row_weights | None, row_layout | None, clamp, stream) -> (status, dx, h, d_row_weights | None)
PyObject* swiglu_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 7, [&]() -> NewTensors {
        const Arg dh(a[0]), q(a[1]), sf(a[2]), w(a[3], true), layout(a[4], true);
        const float clamp = real(a[5]);
        void* stream = pointer<void>(a[6]);
        const at::Tensor& like = tensor(a[0]);
        const bool matrix = dh.d.ndim == 2;
        const int64_t m = matrix ? dh.d.sizes[0] : 0, i = matrix ? dh.d.sizes[1] : 0;
        at::Tensor dx, h, dw;
        unlocked([&] {
            dx = new_matrix(like, m, 2 * i, at::kBFloat16);
            h = new_matrix(like, m, i, at::kBFloat16);
            if (w.given) dw = at::empty({m}, like.options().dtype(at::kFloat));
            return 0;
        });
        Arg ddx, dhh, ddw;
        ddx.fill(dx), dhh.fill(h);
        if (w.given) ddw.fill(dw), ddw.given = true;
        return {call(g_entry.swiglu_backward, dh.get(), q.get(), sf.get(), w.get(), layout.get(), clamp, &ddx.d, &dhh.d,
                     ddw.get(), stream),
                {dx, h, dw}};
    });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<init>("init"),     method<gemm_nt>("gemm_nt"), method<contiguous>("contiguous"),
                           method<masked>("masked"), method<cast>("cast"),       method<dispatch>("dispatch"),
                           method<swiglu>("swiglu"), method<contiguous_swiglu>("contiguous_swiglu"),
                           method<masked_swiglu>("masked_swiglu"),               method<combine>("combine"),
                           method<init_bf16>("init_bf16"), method<m_grouped_ragged>("m_grouped_ragged"),
                           method<k_grouped_ragged>("k_grouped_ragged"),
                           method<swiglu_checkpoint>("swiglu_checkpoint"),
                           method<swiglu_backward>("swiglu_backward"),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_dgbind", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dgbind() { return PyModule_Create(&g_module); }
