// hk_torch.cpp -- attention_forward / attention_backward and the operators round them over torch tensors, from native code:
// reads the tensors, allocates the outputs that were not given, fills the argument block and calls the library.
//
// The two calls on a small problem are host-bound: filling the ctypes blocks, allocating through torch's Python API and
// asking for the current stream took longer than the kernels run.  This module does the same work without Python
// objects in between.  The library is the one attention.py loads (dlsym on its handle), so an instrumented build given
// by HK_ATTENTION_LIB is used here too.
#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <string.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/hk_attention.h"

namespace {

typedef int (*FwdFn)(const hk_attn_fwd_params*, void*);
typedef int (*BwdFn)(const hk_attn_bwd_params*, void*);
typedef int (*ZeroFn)(const hk_attn_bwd_params*, void*);
typedef size_t (*FwdSizeFn)(const hk_attn_fwd_params*);
typedef size_t (*BwdSizeFn)(const hk_attn_bwd_params*);
typedef int (*QkFn)(const hk_qk_params*, void*);
typedef size_t (*QkSizeFn)(const hk_qk_params*);
typedef int (*PrefixFn)(const hk_shared_prefix_params*, void*);
typedef size_t (*PrefixSizeFn)(const hk_shared_prefix_params*);
struct Library {
    FwdFn forward;
    BwdFn backward;
    ZeroFn zero_dq;
    FwdSizeFn fwd_bytes;
    BwdSizeFn bwd_bytes;
    QkFn qk[4];
    QkSizeFn qk_bytes;
    PrefixFn prefix;
    PrefixSizeFn prefix_bytes;
} g_lib = {};

// A tensor argument; None, where it may be left out, gives nullptr.  Anything else is refused: a mask or an output buffer
// of another kind must not pass for one that was not given.  False with TypeError set.
struct TensorArg {
    PyObject* object;
    const char* name;
    bool optional;
    const at::Tensor** tensor;
};
bool tensors(std::initializer_list<TensorArg> args) {
    for (const TensorArg& x : args) {
        *x.tensor = nullptr;
        if (THPVariable_Check(x.object)) {
            *x.tensor = &THPVariable_Unpack(x.object);
        } else if (!x.optional || x.object != Py_None) {
            PyErr_Format(PyExc_TypeError, "%s: expected a tensor%s, not %s", x.name, x.optional ? " or None" : "",
                         Py_TYPE(x.object)->tp_name);
            return false;
        }
    }
    return true;
}

bool refuse(const char* name, const char* what) {
    PyErr_Format(PyExc_AssertionError, "%s: %s", name, what);
    return false;
}

// Whether the attention kernels, which take every tensor for fp32 of the sizes that Q and K give, stay inside this one: of that type,
// and no smaller.  rows: [B, H, T, 64], whose strides have been looked at; otherwise [B, H, T], a number to a row.
// False with AssertionError set.
bool holds(const at::Tensor& t, const char* name, int64_t B, int64_t H, int64_t T, bool rows = true) {
    if (t.scalar_type() != at::kFloat) return refuse(name, "expected float32");
    const at::IntArrayRef size = t.sizes();
    if (!rows && (size.size() < 3 || (T > 1 && t.stride(2) != 1))) return refuse(name, "expected [B,H,T] with unit last stride");
    if (size[0] < B || size[1] < H || size[2] < T) return refuse(name, "smaller than the other tensors");
    return true;
}
// The same for a dense dropout mask, which is read as [B * H, Tq, Tk] without gaps where the call drops anything by it.
bool mask_holds(const at::Tensor* mask, float p, uint32_t flags, int64_t B, int64_t H, int64_t Tq, int64_t Tk) {
    if (!mask || !(p > 0.f) || (flags & HK_FLAG_PHILOX_DROPOUT)) return true;
    if (mask->scalar_type() != at::kFloat || !mask->is_contiguous()) return refuse("dropout_mask", "expected float32, contiguous");
    if ((double)mask->numel() < (double)B * H * Tq * Tk) return refuse("dropout_mask", "smaller than the other tensors");
    return true;
}

// strides of a [B, H, T, 64] view into the block's (B, M, H) triple; false with AssertionError set
bool strides(const at::Tensor& t, int64_t* sB, int64_t* sM, int64_t* sH) {
    if (t.dim() != 4 || t.size(3) != 64 || t.stride(3) != 1) {
        PyErr_SetString(PyExc_AssertionError, "expected [B,H,T,64] with unit last stride");
        return false;
    }
    *sB = t.stride(0);
    *sM = t.stride(2);
    *sH = t.stride(1);
    return true;
}

void* stream_of(PyObject* o) {
    if (o == Py_None) return c10::cuda::getCurrentCUDAStream().stream();
    return reinterpret_cast<void*>(PyLong_AsUnsignedLongLongMask(o));
}

// Runs an entry point's body.  A C++ exception thrown anywhere in it (no device, no memory, a tensor without strides or
// data) becomes the Python exception torch raises for it; left to itself it would end the process.
template <class F>
PyObject* guarded(F&& body) {
    try {
        return body();
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// The interpreter is free for other threads while this lives; it is taken back on every way out.
struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

float* data(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

// workspace: 256-byte aligned start inside a tensor a caller brought; false with AssertionError set if `need` does not fit
bool given_workspace(const at::Tensor* t, size_t need, void** ptr, size_t* bytes) {
    if (!t) return true;
    uint8_t* base = static_cast<uint8_t*>(t->data_ptr());
    const size_t off = (256 - (reinterpret_cast<uintptr_t>(base) & 255u)) & 255u;
    const size_t have = t->nbytes();  // of its elements, whatever type they have
    if (need > 0 && !t->is_contiguous()) return refuse("workspace", "expected contiguous memory");  // an expanded one has less than that
    if (need > 0 && have < off + need) {
        PyErr_SetString(PyExc_AssertionError, "workspace too small");
        return false;
    }
    *ptr = base + off;
    *bytes = have > off ? have - off : 0;
    return true;
}

}  // namespace

// forward(Q, K, V, scale, causal, dropout_p, dropout_mask, seed, offset, q_pos0, k_pos0, bh_pos0, flags, workspace, out,
//         lse, stream) -> (O, LSE), or the negative status of the call
static PyObject* forward_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 17) {
        PyErr_SetString(PyExc_TypeError, "forward: 17 arguments");
        return nullptr;
    }
    const at::Tensor *Q, *K, *V, *mask, *ws, *out, *lse;
    if (!tensors({{a[0], "Q", false, &Q}, {a[1], "K", false, &K}, {a[2], "V", false, &V}, {a[6], "dropout_mask", true, &mask},
                  {a[13], "workspace", true, &ws}, {a[14], "out", true, &out}, {a[15], "lse", true, &lse}}))
        return nullptr;
    hk_attn_fwd_params p = {};
    if (!strides(*Q, &p.q_strideB, &p.q_strideM, &p.q_strideH) || !strides(*K, &p.k_strideB, &p.k_strideM, &p.k_strideH) ||
        !strides(*V, &p.v_strideB, &p.v_strideM, &p.v_strideH))
        return nullptr;
    const int64_t B = Q->size(0), H = Q->size(1), Tq = Q->size(2), Tk = K->size(2);
    const auto opt = Q->options().dtype(at::kFloat);
    at::Tensor O = out ? *out : at::empty({B, H, Tq, 64}, opt);
    at::Tensor L = lse ? *lse : at::empty({B, H, Tq}, opt);
    if (!strides(O, &p.o_strideB, &p.o_strideM, &p.o_strideH)) return nullptr;
    p.lse_strideB = L.stride(0);
    p.lse_strideH = L.stride(1);
    p.Q = data(*Q); p.K = data(*K); p.V = data(*V); p.O = data(O); p.LSE = data(L);
    p.B = (int)B; p.nh = (int)H; p.T = Tq;
    p.scale = (float)PyFloat_AsDouble(a[3]);
    p.is_causal = PyObject_IsTrue(a[4]) != 0;
    p.dropout_p = (float)PyFloat_AsDouble(a[5]);
    p.dropout_mask = mask ? data(*mask) : nullptr;
    p.kv_len = Tk != Tq ? Tk : 0;
    if (a[7] != Py_None) {  // the offset counts only beside a seed
        p.dropout_seed = PyLong_AsUnsignedLongLongMask(a[7]);
        p.dropout_offset = PyLong_AsUnsignedLongLongMask(a[8]);
    }
    p.q_pos0 = PyLong_AsLongLong(a[9]);
    p.k_pos0 = PyLong_AsLongLong(a[10]);
    p.bh_pos0 = (uint32_t)PyLong_AsUnsignedLongLongMask(a[11]);
    p.flags = (uint32_t)PyLong_AsUnsignedLongLongMask(a[12]);
    void* stream = stream_of(a[16]);
    if (PyErr_Occurred()) return nullptr;
    if (!holds(*Q, "Q", B, H, Tq) || !holds(*K, "K", B, H, Tk) || !holds(*V, "V", B, H, Tk) || !holds(O, "out", B, H, Tq) ||
        !holds(L, "lse", B, H, Tq, false) || !mask_holds(mask, p.dropout_p, p.flags, B, H, Tq, Tk))
        return nullptr;
    if (ws && !given_workspace(ws, g_lib.fwd_bytes(&p), &p.workspace, &p.workspace_bytes)) return nullptr;
    int rc;
    {
        NoGil nogil;
        rc = g_lib.forward(&p, stream);
    }
    if (rc != 0) return PyLong_FromLong(rc);
    PyObject* res = PyTuple_New(2);
    if (!res) return nullptr;
    PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(std::move(O)));
    PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(std::move(L)));
    return res;
}

// backward(Q, K, V, O, dO, LSE, scale, causal, dropout_p, dropout_mask, seed, offset, q_pos0, k_pos0, bh_pos0, flags,
//          workspace, D, dQ, dK, dV, stream) -> (dQ, dK, dV, D), or the negative status of the call
static PyObject* backward_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 22) {
        PyErr_SetString(PyExc_TypeError, "backward: 22 arguments");
        return nullptr;
    }
    const at::Tensor *Q, *K, *V, *O, *dO, *LSE, *mask, *ws, *given[4];  // given: dQ, dK, dV, D
    if (!tensors({{a[0], "Q", false, &Q}, {a[1], "K", false, &K}, {a[2], "V", false, &V}, {a[3], "O", true, &O}, {a[4], "dO", false, &dO},
                  {a[5], "LSE", false, &LSE}, {a[9], "dropout_mask", true, &mask}, {a[16], "workspace", true, &ws},
                  {a[17], "D", true, &given[3]}, {a[18], "dQ", true, &given[0]}, {a[19], "dK", true, &given[1]}, {a[20], "dV", true, &given[2]}}))
        return nullptr;
    hk_attn_bwd_params p = {};
    if (!strides(*Q, &p.q_strideB, &p.q_strideM, &p.q_strideH) || !strides(*K, &p.k_strideB, &p.k_strideM, &p.k_strideH) ||
        !strides(*V, &p.v_strideB, &p.v_strideM, &p.v_strideH) || !strides(*dO, &p.do_strideB, &p.do_strideM, &p.do_strideH) ||
        (O && !strides(*O, &p.o_strideB, &p.o_strideM, &p.o_strideH)))
        return nullptr;
    const int64_t B = Q->size(0), H = Q->size(1), Tq = Q->size(2), Tk = K->size(2);
    p.flags = (uint32_t)PyLong_AsUnsignedLongLongMask(a[15]);
    p.B = (int)B; p.nh = (int)H; p.T = (int)Tq;
    p.kv_len = Tk != Tq ? Tk : 0;
    void* stream = stream_of(a[21]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor r[4], slabs;  // dQ, dK, dV, D
    const auto opt = Q->options().dtype(at::kFloat);
    for (int i = 0; i < 4; ++i)
        r[i] = given[i] ? *given[i] : i == 3 ? at::empty({B, H, Tq}, opt) : at::empty({B, H, i == 0 ? Tq : Tk, 64}, opt);
    if (!strides(r[0], &p.dq_strideB, &p.dq_strideM, &p.dq_strideH) || !strides(r[1], &p.dk_strideB, &p.dk_strideM, &p.dk_strideH) ||
        !strides(r[2], &p.dv_strideB, &p.dv_strideM, &p.dv_strideH))
        return nullptr;
    p.d_strideB = r[3].stride(0);
    p.d_strideH = r[3].stride(1);
    p.lse_strideB = LSE->stride(0);
    p.lse_strideH = LSE->stride(1);
    if (ws) {
        if (!given_workspace(ws, g_lib.bwd_bytes(&p), &p.workspace, &p.workspace_bytes)) return nullptr;
    } else if (p.flags & HK_FLAG_DETERMINISTIC_DQ) {  // the slabs of partial dQ are the only scratch there is
        hk_attn_bwd_params q = p;
        q.flags |= HK_FLAG_OPERANDS_PREROUNDED;
        const size_t bytes = g_lib.bwd_bytes(&q);
        // They are given back when this call returns, long before the kernels are done with them: they have to come from
        // the pool of the stream the kernels run on, where the next user of the memory is behind these.
        c10::cuda::OptionalCUDAStreamGuard guard;
        if (a[21] != Py_None && Q->is_cuda()) {
            const cudaStream_t s = static_cast<cudaStream_t>(stream);
            const auto device = Q->device().index();
            // 0 and cudaStreamLegacy are the default stream, which torch does not know by a handle
            guard.reset_stream(s == nullptr || s == cudaStreamLegacy ? c10::cuda::getDefaultCUDAStream(device)
                                                                     : c10::cuda::getStreamFromExternal(s, device));
        }
        slabs = at::empty({(int64_t)bytes + 256}, Q->options().dtype(at::kByte));
        if (!given_workspace(&slabs, bytes, &p.workspace, &p.workspace_bytes)) return nullptr;
    }
    p.Q = data(*Q); p.K = data(*K); p.V = data(*V); p.O = O ? data(*O) : nullptr; p.dO = data(*dO); p.LSE = data(*LSE);
    p.dQ = data(r[0]); p.dK = data(r[1]); p.dV = data(r[2]); p.D = data(r[3]);
    p.scale = (float)PyFloat_AsDouble(a[6]);
    p.is_causal = PyObject_IsTrue(a[7]) != 0;
    p.dropout_p = (float)PyFloat_AsDouble(a[8]);
    p.dropout_mask = mask ? data(*mask) : nullptr;
    if (a[10] != Py_None) {  // the offset counts only beside a seed
        p.dropout_seed = PyLong_AsUnsignedLongLongMask(a[10]);
        p.dropout_offset = PyLong_AsUnsignedLongLongMask(a[11]);
    }
    p.q_pos0 = PyLong_AsLongLong(a[12]);
    p.k_pos0 = PyLong_AsLongLong(a[13]);
    p.bh_pos0 = (uint32_t)PyLong_AsUnsignedLongLongMask(a[14]);
    if (PyErr_Occurred()) return nullptr;
    if (!holds(*Q, "Q", B, H, Tq) || !holds(*K, "K", B, H, Tk) || !holds(*V, "V", B, H, Tk) || (O && !(p.flags & HK_FLAG_D_PRECOMPUTED) && !holds(*O, "O", B, H, Tq)) ||
        !holds(*dO, "dO", B, H, Tq) || !holds(*LSE, "LSE", B, H, Tq, false) || !holds(r[0], "dQ", B, H, Tq) || !holds(r[1], "dK", B, H, Tk) ||
        !holds(r[2], "dV", B, H, Tk) || !holds(r[3], "D", B, H, Tq, false) || !mask_holds(mask, p.dropout_p, p.flags, B, H, Tq, Tk))
        return nullptr;
    int rc;
    {
        NoGil nogil;
        rc = g_lib.backward(&p, stream);
    }
    if (rc != 0) return PyLong_FromLong(rc);
    PyObject* res = PyTuple_New(4);
    if (!res) return nullptr;
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(res, i, THPVariable_Wrap(std::move(r[i])));
    return res;
}

// zero(x, stream) -> status: zeroes a [B, H, T, 64] view
static PyObject* zero_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "zero: 2 arguments");
        return nullptr;
    }
    const at::Tensor* x;
    if (!tensors({{a[0], "dQ", false, &x}})) return nullptr;
    hk_attn_bwd_params p = {};
    if (!strides(*x, &p.dq_strideB, &p.dq_strideM, &p.dq_strideH)) return nullptr;
    p.B = (int)x->size(0); p.nh = (int)x->size(1); p.T = (int)x->size(2);
    p.dQ = data(*x);
    void* stream = stream_of(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (!holds(*x, "dQ", 0, 0, 0)) return nullptr;
    return PyLong_FromLong(g_lib.zero_dq(&p, stream));
}

// ---- the operators round the attention: tensors of three types, on one device, checked against each other -------------------
namespace {

int dtype_code(const at::Tensor& t) {
    return t.scalar_type() == at::kFloat ? HK_F32 : t.scalar_type() == at::kBFloat16 ? HK_BF16 : t.scalar_type() == at::kHalf ? HK_F16 : -1;
}
at::ScalarType scalar_of(int code) { return code == HK_BF16 ? at::kBFloat16 : code == HK_F16 ? at::kHalf : at::kFloat; }

constexpr int64_t MOST = 1 << 30;  // rows, heads, batches: what the argument blocks' integers hold

// t as [B, n, T, 64] of `type` (-1: of any of the three) into a block's view; the sizes that are -1 are not looked at.
// alone: as [n, T, 64] too, a batch of one.
bool view(const at::Tensor& t, const char* name, int64_t B, int64_t n, int64_t T, int type, hk_view* v, bool alone = false) {
    const at::IntArrayRef size = t.sizes(), stride = t.strides();
    const int lead = alone && t.dim() == 3 ? 0 : 1;  // the dimension of the heads
    if (t.dim() != lead + 3 || size[lead + 2] != 64 || stride[lead + 2] != 1) return refuse(name, "expected [B,H,T,64] with unit last stride");
    for (int i = 0; i < lead + 2; ++i)
        if (size[i] > MOST) return refuse(name, "too large");
    if ((B >= 0 && (lead ? size[0] : 1) != B) || (n >= 0 && size[lead] != n) || (T >= 0 && size[lead + 1] != T)) return refuse(name, "sizes do not fit the other tensors'");
    if (dtype_code(t) < 0 || (type >= 0 && dtype_code(t) != type))
        return refuse(name, type < 0 ? "expected float32, bfloat16 or float16" : "element type does not fit the other tensors'");
    *v = {t.data_ptr(), lead ? stride[0] : 0, stride[lead + 1], stride[lead]};
    return true;
}

// All of them on one CUDA device; false with AssertionError set.
bool one_device(std::initializer_list<const at::Tensor*> all) {
    const at::Tensor* first = nullptr;
    for (const at::Tensor* t : all) {
        if (!t) continue;
        if (!first) first = t;
        if (!t->is_cuda()) return refuse("tensors", "expected CUDA tensors");
        if (t->device() != first->device()) return refuse("tensors", "expected all on one device");
    }
    return true;
}

// A tensor that a kernel is about to fill, without the way through the dispatcher, which takes as long again as the allocation;
// torch's own switch that fills such tensors is heard.  Each result has memory of its own: two in one allocation would take 0.4 us
// less, but who keeps or writes out one of them would have both.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
    if (at::globalContext().deterministicAlgorithms() && at::globalContext().deterministicFillUninitializedMemory())
        return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// Makes the tensors' device the current one and the stream asked for (None: that device's current one) the one that
// results and workspaces are allocated for: they are written there, whatever becomes of them here.
struct OnStream {
    c10::cuda::CUDAGuard device;
    c10::cuda::OptionalCUDAStreamGuard guard;
    void* stream;
    OnStream(PyObject* o, const at::Tensor& t) : device(t.device()) {
        stream = stream_of(o);
        if (o == Py_None || PyErr_Occurred()) return;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        // 0 and cudaStreamLegacy are the default stream, which torch does not know by a handle
        guard.reset_stream(s == nullptr || s == cudaStreamLegacy ? c10::cuda::getDefaultCUDAStream(t.device().index())
                                                                 : c10::cuda::getStreamFromExternal(s, t.device().index()));
    }
};

PyObject* wrap(std::initializer_list<at::Tensor> r) {
    PyObject* res = PyTuple_New((Py_ssize_t)r.size());
    if (!res) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& t : r) {
        PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
        PyTuple_SET_ITEM(res, i++, o);
    }
    return res;
}

}  // namespace

// qk(which, Q, K, dQ, dK, w_q, w_k, positions, plan, eps, out_dtype, out_q, out_k, stream)
//   which: 0 rotation, 1 its backward, 2 norm and rotation, 3 its backward; plan: the bytes of an hk_rotary_plan;
//   out_dtype: of the results of 0, 1, 2 (hk_dtype, -1: the argument's)
// -> the results, with 3 followed by the weights' gradients, or the negative status of the call
static PyObject* qk_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 14) {
        PyErr_SetString(PyExc_TypeError, "qk: 14 arguments");
        return nullptr;
    }
    const int which = (int)PyLong_AsLong(a[0]);
    if (PyErr_Occurred()) return nullptr;
    if (which < 0 || which > 3) {
        PyErr_SetString(PyExc_ValueError, "qk: which");
        return nullptr;
    }
    const bool norm = which >= 2, back = which & 1, grads = back, rows = which != 1;
    const at::Tensor *x[2], *g[2], *w[2], *pos, *out[2];
    if (!tensors({{a[1], "Q", !rows, &x[0]}, {a[2], "K", true, &x[1]}, {a[3], "dQ", !grads, &g[0]}, {a[4], "dK", true, &g[1]},
                  {a[5], "w_q", true, &w[0]}, {a[6], "w_k", true, &w[1]}, {a[7], "positions", false, &pos},
                  {a[11], "out_q", true, &out[0]}, {a[12], "out_k", true, &out[1]}}))
        return nullptr;
    hk_qk_params p = {};
    if (!PyBytes_Check(a[8]) || PyBytes_GET_SIZE(a[8]) != (Py_ssize_t)sizeof(p.plan)) {
        PyErr_SetString(PyExc_TypeError, "plan: expected the bytes of a plan");
        return nullptr;
    }
    memcpy(&p.plan, PyBytes_AS_STRING(a[8]), sizeof(p.plan));
    p.eps = (float)PyFloat_AsDouble(a[9]);
    int out_type = (int)PyLong_AsLong(a[10]);
    if (PyErr_Occurred()) return nullptr;

    const at::Tensor** src = rows ? x : g;  // what decides sizes
    const char* names[2][2] = {{"Q", "K"}, {"dQ", "dK"}};
    if (rows && grads && !x[1] != !g[1]) return refuse("dK", "expected together with K"), nullptr;
    hk_view none = {}, *src_view[2] = {rows ? &p.q : &p.dq_out, rows ? &p.k : &p.dk_out};
    if (!view(*src[0], names[!rows][0], -1, -1, -1, -1, src_view[0])) return nullptr;
    const int64_t B = src[0]->size(0), H = src[0]->size(1), T = src[0]->size(2), Hk = src[1] ? src[1]->size(1) : 0;
    const int type = dtype_code(*src[0]);
    if (src[1] && !view(*src[1], names[!rows][1], B, -1, T, type, src_view[1])) return nullptr;
    p.B = (int)B; p.nh = (int)H; p.nh_k = (int)Hk; p.T = T;
    if (which == 3) {  // the gradients' type stands for out_dtype, the results are of the rows' type
        if (!view(*g[0], "dQ", B, H, T, -1, &p.dq_out)) return nullptr;
        p.out_dtype = dtype_code(*g[0]);
        if (g[1] && !view(*g[1], "dK", B, Hk, T, p.out_dtype, &p.dk_out)) return nullptr;
        p.dtype = type;
        out_type = type;
    } else {
        if (out_type < 0) out_type = out[0] ? dtype_code(*out[0]) : type;
        p.dtype = back ? out_type : type;
        p.out_dtype = back ? type : out_type;
    }
    for (int k = 0; k < 2; ++k) {
        const char* name = k ? "w_k" : "w_q";
        if (!norm || !w[k]) continue;
        if (w[k]->dim() != 1 || w[k]->size(0) != 64 || w[k]->stride(0) != 1) return refuse(name, "expected [64], contiguous"), nullptr;
        if (dtype_code(*w[k]) < 0 || (k && w[0] && dtype_code(*w[0]) != dtype_code(*w[k])))
            return refuse(name, "element type does not fit the other tensors'"), nullptr;
        p.weight_dtype = dtype_code(*w[k]);
    }
    if (pos->dim() != 3 || pos->size(0) != p.plan.n_axes || pos->size(1) != B || pos->size(2) != T)
        return refuse("positions", "expected [axes,B,T]"), nullptr;
    if (pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong) return refuse("positions", "expected int32 or int64"), nullptr;
    hk_view* dst_view[2] = {back ? &p.dq : &p.q_out, back ? &p.dk : &p.k_out};
    for (int k = 0; k < 2; ++k) {
        if (!out[k]) continue;
        if (!src[k]) return refuse("out_k", "there is no K"), nullptr;
        if (!view(*out[k], k ? "out_k" : "out_q", B, k ? Hk : H, T, out_type, &none)) return nullptr;
    }
    if (!one_device({src[0], src[1], x[0], x[1], g[0], g[1], norm ? w[0] : nullptr, norm ? w[1] : nullptr, pos, out[0], out[1]})) return nullptr;
    OnStream on(a[13], *src[0]);
    if (PyErr_Occurred()) return nullptr;

    const at::Device device = src[0]->device();
    at::Tensor r[2], dw[2], ws;
    for (int k = 0; k < 2; ++k) {
        if (!src[k]) continue;
        r[k] = out[k] ? *out[k] : fresh({B, k ? Hk : H, T, 64}, scalar_of(out_type), device);
        *dst_view[k] = {r[k].data_ptr(), r[k].stride(0), r[k].stride(2), r[k].stride(1)};
    }
    p.q_weight = norm && w[0] ? w[0]->data_ptr() : nullptr;
    p.k_weight = norm && w[1] ? w[1]->data_ptr() : nullptr;
    if (which == 3) {
        for (int k = 0; k < 2; ++k)
            if (w[k] && src[k]) dw[k] = fresh({64}, at::kFloat, device);
        p.dq_weight = dw[0].defined() ? data(dw[0]) : nullptr;
        p.dk_weight = dw[1].defined() ? data(dw[1]) : nullptr;
        p.workspace_bytes = g_lib.qk_bytes(&p);
        ws = fresh({(int64_t)p.workspace_bytes}, at::kByte, device);
        p.workspace = ws.data_ptr();
    }
    p.positions = pos->data_ptr();
    p.pos_bits = pos->scalar_type() == at::kLong ? 64 : 32;
    p.pos_strideA = pos->stride(0); p.pos_strideB = pos->stride(1); p.pos_strideT = pos->stride(2);
    int rc;
    {
        NoGil nogil;
        rc = g_lib.qk[which](&p, on.stream);
    }
    if (rc != 0) return PyLong_FromLong(rc);
    return which == 3 ? wrap({r[0], r[1], dw[0], dw[1]}) : wrap({r[0], r[1]});
}

// What of a shared prefix's call its workspace depends on; false with AssertionError set.
static bool prefix_sizes(const at::Tensor& Q, const at::Tensor& K_prefix, const at::Tensor& K, hk_shared_prefix_params* p) {
    if (!view(Q, "Q", -1, -1, -1, -1, &p->Q)) return false;
    p->dtype = dtype_code(Q);
    if (!view(K, "K", Q.size(0), -1, -1, p->dtype, &p->K) || !view(K_prefix, "K_prefix", 1, K.size(1), -1, p->dtype, &p->Kp, true)) return false;
    p->B = (int)Q.size(0); p->nh = (int)Q.size(1); p->nh_kv = (int)K.size(1);
    p->T = Q.size(2); p->prefix_len = K_prefix.size(-2); p->kv_len = K.size(2);
    return true;
}

// prefix_workspace(Q, K_prefix, K) -> bytes that are enough for the workspace of the call, wherever they start
static PyObject* prefix_workspace_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "prefix_workspace: 3 arguments");
        return nullptr;
    }
    const at::Tensor *Q, *K_prefix, *K;
    if (!tensors({{a[0], "Q", false, &Q}, {a[1], "K_prefix", false, &K_prefix}, {a[2], "K", false, &K}})) return nullptr;
    hk_shared_prefix_params p = {};
    if (!prefix_sizes(*Q, *K_prefix, *K, &p)) return nullptr;
    p.scale = 1.f;
    c10::cuda::OptionalCUDAGuard device;  // the plan goes by its SMs
    if (Q->is_cuda()) device.set_device(Q->device());
    const size_t need = g_lib.prefix_bytes(&p);
    return PyLong_FromSize_t(need > 0 ? need + 256 : 0);
}

// prefix(Q, K_prefix, V_prefix, K, V, lengths, scale, causal, workspace, out, lse, stream) -> (O, LSE), or the negative status
static PyObject* prefix_body(PyObject* const* a, Py_ssize_t n) {
    if (n != 12) {
        PyErr_SetString(PyExc_TypeError, "prefix: 12 arguments");
        return nullptr;
    }
    const at::Tensor *Q, *kv[4], *lens, *ws, *out, *lse;
    if (!tensors({{a[0], "Q", false, &Q}, {a[1], "K_prefix", false, &kv[0]}, {a[2], "V_prefix", false, &kv[1]}, {a[3], "K", false, &kv[2]},
                  {a[4], "V", false, &kv[3]}, {a[5], "lengths", true, &lens}, {a[8], "workspace", true, &ws}, {a[9], "out", true, &out}, {a[10], "lse", true, &lse}}))
        return nullptr;
    hk_shared_prefix_params p = {};
    if (!prefix_sizes(*Q, *kv[0], *kv[2], &p)) return nullptr;
    const int64_t B = Q->size(0), H = Q->size(1), T = Q->size(2), Hk = kv[2]->size(1);
    if (!view(*kv[3], "V", B, Hk, p.kv_len, p.dtype, &p.V) || !view(*kv[1], "V_prefix", 1, Hk, p.prefix_len, p.dtype, &p.Vp, true)) return nullptr;
    if (lens && (lens->dim() != 1 || lens->size(0) != B || (B > 1 && lens->stride(0) != 1) || lens->scalar_type() != at::kInt))
        return refuse("lengths", "expected [B] of int32, contiguous"), nullptr;
    if (out && !view(*out, "out", B, H, T, p.dtype, &p.O)) return nullptr;
    if (lse && (lse->dim() != 3 || lse->size(0) != B || lse->size(1) != H || lse->size(2) != T || (T > 1 && lse->stride(2) != 1) || lse->scalar_type() != at::kFloat))
        return refuse("lse", "expected [B,H,T] of float32 with unit last stride"), nullptr;
    p.scale = (float)PyFloat_AsDouble(a[6]);
    p.is_causal = PyObject_IsTrue(a[7]) != 0;
    if (PyErr_Occurred()) return nullptr;
    p.lengths = lens ? static_cast<const int32_t*>(lens->data_ptr()) : nullptr;
    if (!one_device({Q, kv[0], kv[1], kv[2], kv[3], lens, ws, out, lse})) return nullptr;
    OnStream on(a[11], *Q);
    if (PyErr_Occurred()) return nullptr;
    const at::Device device = Q->device();
    at::Tensor O = out ? *out : fresh({B, H, T, 64}, scalar_of(p.dtype), device), L = lse ? *lse : fresh({B, H, T}, at::kFloat, device), own;
    p.O = {O.data_ptr(), O.stride(0), O.stride(2), O.stride(1)};
    p.LSE = data(L); p.lse_strideB = L.stride(0); p.lse_strideH = L.stride(1);
    const size_t need = g_lib.prefix_bytes(&p);
    if (!ws && need > 0) {
        own = fresh({(int64_t)need + 256}, at::kByte, device);
        ws = &own;
    }
    if (ws && !given_workspace(ws, need, &p.workspace, &p.workspace_bytes)) return nullptr;
    int rc;
    {
        NoGil nogil;
        rc = g_lib.prefix(&p, on.stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : wrap({O, L});
}

static PyObject* qk(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return qk_body(a, n); }); }
static PyObject* prefix(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return prefix_body(a, n); }); }
static PyObject* prefix_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return prefix_workspace_body(a, n); }); }

static PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return forward_body(a, n); }); }
static PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return backward_body(a, n); }); }
static PyObject* zero(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded([&] { return zero_body(a, n); }); }

// bind(handle): the dlopen handle of libhk_attention.so
static PyObject* bind(PyObject*, PyObject* h) {
    void* so = reinterpret_cast<void*>(PyLong_AsUnsignedLongLongMask(h));
    if (PyErr_Occurred()) return nullptr;
    g_lib.forward = reinterpret_cast<FwdFn>(dlsym(so, "hk_attn_forward_noscratch"));
    g_lib.backward = reinterpret_cast<BwdFn>(dlsym(so, "hk_attn_backward_noscratch"));
    g_lib.zero_dq = reinterpret_cast<ZeroFn>(dlsym(so, "hk_attn_zero_dq"));
    g_lib.fwd_bytes = reinterpret_cast<FwdSizeFn>(dlsym(so, "hk_attn_fwd_workspace_bytes"));
    g_lib.bwd_bytes = reinterpret_cast<BwdSizeFn>(dlsym(so, "hk_attn_bwd_workspace_bytes"));
    const char* qk_names[4] = {"hk_rotary_forward", "hk_rotary_backward", "hk_qk_norm_rotary_forward", "hk_qk_norm_rotary_backward"};
    bool all = true;
    for (int i = 0; i < 4; ++i) all = (g_lib.qk[i] = reinterpret_cast<QkFn>(dlsym(so, qk_names[i]))) && all;
    g_lib.qk_bytes = reinterpret_cast<QkSizeFn>(dlsym(so, "hk_qk_norm_rotary_workspace_bytes"));
    g_lib.prefix = reinterpret_cast<PrefixFn>(dlsym(so, "hk_shared_prefix_attention"));
    g_lib.prefix_bytes = reinterpret_cast<PrefixSizeFn>(dlsym(so, "hk_shared_prefix_workspace_bytes"));
    if (!all || !g_lib.qk_bytes || !g_lib.prefix || !g_lib.prefix_bytes || !g_lib.forward || !g_lib.backward || !g_lib.zero_dq || !g_lib.fwd_bytes || !g_lib.bwd_bytes) {
        PyErr_SetString(PyExc_ImportError, "libhk_attention.so lacks an entry point");
        return nullptr;
    }
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(backward)), METH_FASTCALL, nullptr},
    {"zero", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(zero)), METH_FASTCALL, nullptr},
    {"qk", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk)), METH_FASTCALL, nullptr},
    {"prefix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefix)), METH_FASTCALL, nullptr},
    {"prefix_workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefix_workspace)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

PyMODINIT_FUNC PyInit__hk_torch() { return PyModule_Create(&module); }
