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
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
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
    decltype(&dg_moe_dispatch_max_rows) dispatch_max_rows;
    decltype(&dg_moe_dispatch_workspace_size) dispatch_workspace_size;
    decltype(&dg_moe_dispatch_backward) dispatch_backward;
    decltype(&dg_moe_combine_backward) combine_backward;
    decltype(&dg_per_token_cast_to_fp4) cast4;
    decltype(&dg_cast_back_from_fp4) cast_back4;
    decltype(&dg_m_grouped_fp4_gemm_nt_ragged) ragged_fp4;
    decltype(&dg_fp4_gemm_ragged_workspace_size) ragged_fp4_workspace_size;
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

// init_rows(addresses of the entry points after those)
PyObject* init_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        auto set = [&](auto& entry, int i) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(pointer<void>(a[i])); };
        set(g_entry.dispatch_max_rows, 0), set(g_entry.dispatch_workspace_size, 1);
        set(g_entry.dispatch_backward, 2), set(g_entry.combine_backward, 3);
        set(g_entry.cast4, 4), set(g_entry.cast_back4, 5);
        set(g_entry.ragged_fp4, 6), set(g_entry.ragged_fp4_workspace_size, 7);
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
    Workspace(int form, const at::Tensor& out, int64_t rows, int64_t m, int64_t n, int64_t k, int64_t groups)
        : Workspace(out, out.is_cuda() ? g_entry.ragged_workspace_size(form, rows, m, n, k, (int32_t)groups) : 0) {}
    Workspace(const at::Tensor& out, int64_t bytes) {
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

// ragged_fp4(a, a_sf, b, b_sf, d, group_ends, alignment, stream)
PyObject* ragged_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Arg ta(a[0]), sa(a[1]), tb(a[2]), sb(a[3]), d(a[4]), ends(a[5]);
        const int32_t alignment = integer(a[6]);
        void* stream = pointer<void>(a[7]);
        const bool fits = ta.d.ndim == 2 && tb.d.ndim == 3 && tensor(a[4]).is_cuda();
        const Workspace ws(tensor(a[4]), fits ? g_entry.ragged_fp4_workspace_size(ta.d.sizes[0], tb.d.sizes[1], 2 * ta.d.sizes[1],
                                                                                  (int32_t)tb.d.sizes[0]) : 0);
        return call(g_entry.ragged_fp4, ta.get(), sa.get(), tb.get(), sb.get(), d.get(), ends.get(), alignment, ws.arg.get(),
                    stream);
    });
}

// Whether a kernel may stand for torch's operations on a tensor: its memory holds its values (no negative view, no zeros
// without memory), and torch does not have to follow what becomes of it (as a subclass, in a transform of torch.func, with
// a tangent; with a gradient, where one could pass).
bool kernel_may_stand(PyObject* o, bool gradient) {
    const at::Tensor& t = tensor(o);
    constexpr c10::DispatchKeySet followed{c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::Negative,
                                           c10::DispatchKey::ZeroTensor, c10::DispatchKey::FuncTorchBatched,
                                           c10::DispatchKey::FuncTorchGradWrapper};
    return t.is_cuda() && THPVariable_CheckExact(o) && !t.key_set().has_any(followed) && !t._fw_grad(0).defined() &&
           !(gradient && t.requires_grad() && c10::GradMode::is_enabled());
}
// Launches that a 4-bit cast of [m, n] needs: one takes below 2^24 blocks of 4 x 1024 values.
int32_t cast4_launches(int64_t m, int64_t n) {
    const int64_t rows = ((int64_t(1) << 24) - 1) / std::max<int64_t>((n + 1023) / 1024, 1) * 4;
    return m > rows ? 2 : 1;
}

// cast4_takes(x, gran_k, use_ue8m0) -> 0: a call for the torch operations, 1: for the kernel, 2: for it, in several launches
PyObject* cast4_takes(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&] {
        const at::Tensor& x = tensor(a[0]);
        const int32_t gran = integer(a[1]), ue8m0 = integer(a[2]);
        if (x.dim() != 2 || x.scalar_type() != at::kBFloat16 || (gran != 32 && gran != 64 && gran != 128)) return 0;
        // (float scales carry a gradient, codes and power-of-two scales none)
        if (!kernel_may_stand(a[0], !ue8m0) || x.stride(1) != 1 || x.size(1) % 2 != 0 || x.size(1) >= (1 << 27)) return 0;
        return cast4_launches(x.size(0), x.size(1));
    });
}

// cast_back4_takes(q, sf, gran_k, packed) -> as cast4_takes
PyObject* cast_back4_takes(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&] {
        const at::Tensor &q = tensor(a[0]), &sf = tensor(a[1]);
        const int32_t gran = integer(a[2]), packed = integer(a[3]);
        if (q.dim() != 2 || sf.dim() != 2 || q.scalar_type() != at::kChar || (gran != 32 && gran != 64 && gran != 128)) return 0;
        if (sf.scalar_type() != (packed ? at::kInt : at::kFloat) || sf.device() != q.device()) return 0;
        if (!kernel_may_stand(a[0], false) || !kernel_may_stand(a[1], true)) return 0;
        const int64_t m = q.size(0), half = q.size(1), groups = (2 * half + gran - 1) / gran;
        if (half >= (1 << 26) || (half > 1 && q.stride(1) != 1)) return 0;
        if (sf.size(0) != m || sf.size(1) != (packed ? (groups + 3) / 4 : groups)) return 0;
        return cast4_launches(m, 2 * half);
    });
}

// cast4(x, gran_k, use_ue8m0, packed, stream) -> (status, q, sf)
PyObject* cast4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 5, [&]() -> NewTensors {
        const Arg x(a[0]);
        const int32_t gran = integer(a[1]), ue8m0 = integer(a[2]), packed = integer(a[3]);
        void* stream = pointer<void>(a[4]);
        const at::Tensor& like = tensor(a[0]);
        const bool matrix = x.d.ndim == 2 && gran > 0;   // (otherwise the call refuses it)
        const int64_t m = matrix ? x.d.sizes[0] : 0, cols = matrix ? x.d.sizes[1] : 0;
        const int64_t groups = matrix ? (cols + gran - 1) / gran : 0;
        at::Tensor q, sf;
        unlocked([&] {
            q = new_matrix(like, m, cols / 2, at::kChar);
            sf = packed ? new_matrix(like, m, (groups + 3) / 4, at::kInt) : new_matrix(like, m, groups, at::kFloat);
            return 0;
        });
        Arg dq, ds;
        dq.fill(q), ds.fill(sf);
        return {call(g_entry.cast4, x.get(), &dq.d, &ds.d, gran, ue8m0, stream), {q, sf}};
    });
}

// cast_back4(q, sf, gran_k, bf16, stream) -> (status, y)
PyObject* cast_back4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 5, [&]() -> NewTensors {
        const Arg q(a[0]), sf(a[1]);
        const int32_t gran = integer(a[2]), bf16 = integer(a[3]);
        void* stream = pointer<void>(a[4]);
        const at::Tensor& like = tensor(a[0]);
        const bool matrix = q.d.ndim == 2;
        at::Tensor y;
        unlocked([&] {
            y = new_matrix(like, matrix ? q.d.sizes[0] : 0, matrix ? 2 * q.d.sizes[1] : 0, bf16 ? at::kBFloat16 : at::kFloat);
            return 0;
        });
        Arg dy;
        dy.fill(y);
        return {call(g_entry.cast_back4, q.get(), sf.get(), &dy.d, gran, stream), {y}};
    });
}

// dispatch_rows(x, x_sf | None, topk, topk_weights | None, experts, layout, alignment, max_m, out | None, out_sf | None,
//               stream) -> (status, a, sf | None, grouped_layout, pos, row_weights | None)
// (its five to seven allocations here, not in Python)
PyObject* dispatch_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 11, [&]() -> NewTensors {
        const Arg x(a[0]), x_sf(a[1], true), topk(a[2]), topk_w(a[3], true);
        const int32_t experts = integer(a[4]), layout = integer(a[5]), alignment = integer(a[6]), max_m = integer(a[7]);
        const bool given = a[8] != Py_None, given_sf = a[9] != Py_None;
        at::Tensor out = given ? tensor(a[8]) : at::Tensor(), sf = given_sf ? tensor(a[9]) : at::Tensor();
        void* stream = pointer<void>(a[10]);
        const at::Tensor& like = tensor(a[0]);
        if (x.d.ndim != 2 || topk.d.ndim != 2)
            throw std::runtime_error("Assertion error (deep_gemm): x.dim() == 2 and topk_idx.dim() == 2");
        const bool masked = layout == 2;
        const int64_t t = x.d.sizes[0], k = topk.d.sizes[1];
        int64_t rows = masked ? (int64_t)experts * max_m : g_entry.dispatch_max_rows(t, (int32_t)k, experts, alignment);
        if (experts <= 0 || rows < 0)
            throw std::runtime_error("Assertion error (deep_gemm): num_experts > 0, alignment > 0, max_m >= 0 and topk > 0");
        if (given && !masked && out.dim() == 2) rows = out.size(0);   // (at least as many: the call checks it)
        at::Tensor meta, pos, w, ws;
        unlocked([&] {
            auto fresh = [&](int64_t cols, at::ScalarType type) {
                return masked ? at::empty({experts, max_m, cols}, like.options().dtype(type)) : new_matrix(like, rows, cols, type);
            };
            if (!given) out = fresh(x.d.sizes[1], like.scalar_type());
            if (!given_sf && x_sf.given && x_sf.d.ndim == 2) sf = fresh(x_sf.d.sizes[1], x_sf.d.dtype == DG_I32 ? at::kInt : at::kFloat);
            meta = at::empty({layout == 0 ? rows : (int64_t)experts}, like.options().dtype(at::kInt));
            pos = new_matrix(like, t, k, at::kInt);
            if (topk_w.given) w = at::empty({rows}, like.options().dtype(at::kFloat));
            ws = at::empty({std::max<int64_t>(g_entry.dispatch_workspace_size(t, experts) / 4, 1)}, like.options().dtype(at::kInt));
            return 0;
        });
        Arg da, dsf, dm, dp, dw, dws;
        da.fill(out), dm.fill(meta), dp.fill(pos), dws.fill(ws);
        if (sf.defined()) dsf.fill(sf), dsf.given = true;
        if (w.defined()) dw.fill(w), dw.given = true;
        const int32_t status = call(g_entry.dispatch, x.get(), x_sf.get(), topk.get(), topk_w.get(), experts, layout, alignment,
                                    &da.d, dsf.get(), &dm.d, &dp.d, dw.get(), &dws.d, stream);
        if (w.defined() && masked) w = w.view({experts, max_m});
        return {status, {out, sf, meta, pos, w}};
    });
}

// dispatch_backward(drows, pos, drow_weights | None, stream) -> (status, dx, d_topk_weights | None)
PyObject* dispatch_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 4, [&]() -> NewTensors {
        const Arg rows(a[0]), pos(a[1]), w(a[2], true);
        void* stream = pointer<void>(a[3]);
        const at::Tensor& like = tensor(a[0]);
        const bool fits = rows.d.ndim >= 2 && pos.d.ndim == 2;   // (otherwise the call refuses them)
        const int64_t t = fits ? pos.d.sizes[0] : 0, k = fits ? pos.d.sizes[1] : 0;
        at::Tensor dx, dw;
        unlocked([&] {
            dx = new_matrix(like, t, fits ? rows.d.sizes[rows.d.ndim - 1] : 0, at::kBFloat16);
            if (w.given) dw = new_matrix(like, t, k, at::kFloat);
            return 0;
        });
        Arg ddx, ddw;
        ddx.fill(dx);
        if (w.given) ddw.fill(dw), ddw.given = true;
        return {call(g_entry.dispatch_backward, rows.get(), pos.get(), w.get(), &ddx.d, ddw.get(), stream), {dx, dw}};
    });
}

// combine_backward(dout, y, pos, topk_weights | None, dy | None, stream) -> (status, dy, d_topk_weights | None)
PyObject* combine_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded_new(n, 6, [&]() -> NewTensors {
        const Arg dout(a[0]), y(a[1]), pos(a[2]), w(a[3], true);
        const bool given = a[4] != Py_None;
        at::Tensor dy = given ? tensor(a[4]) : at::Tensor(), dw;
        void* stream = pointer<void>(a[5]);
        const at::Tensor& like = tensor(a[1]);
        const bool fits = pos.d.ndim == 2;
        unlocked([&] {
            if (!given) dy = at::zeros(like.sizes(), like.options().dtype(at::kBFloat16));
            if (w.given) dw = new_matrix(like, fits ? pos.d.sizes[0] : 0, fits ? pos.d.sizes[1] : 0, at::kFloat);
            return 0;
        });
        Arg ddy, ddw;
        ddy.fill(dy);
        if (w.given) ddw.fill(dw), ddw.given = true;
        return {call(g_entry.combine_backward, dout.get(), y.get(), pos.get(), w.get(), &ddy.d, ddw.get(), stream), {dy, dw}};
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
                           method<init_rows>("init_rows"), method<ragged_fp4>("ragged_fp4"), method<cast4>("cast4"),
                           method<cast_back4>("cast_back4"), method<cast4_takes>("cast4_takes"),
                           method<cast_back4_takes>("cast_back4_takes"), method<dispatch_rows>("dispatch_rows"),
                           method<dispatch_backward>("dispatch_backward"),
                           method<combine_backward>("combine_backward"),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_dgbind", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dgbind() { return PyModule_Create(&g_module); }
