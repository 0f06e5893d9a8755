// The ordinary call of the operators around the expert layer (grouped routing, residual norm, int8 product) and of those of a
// decode step of a few requests (whole expert layer, low-rank adapters) from tensors to launch in one native call: their
// smallest calls are bound by the host.  In Python the checks and the outputs of one
// take 3 to 5 us beside a launch of 2.8 (small calls: routing 6.5, norm 8.0, product 6.4 us; through this 5.1, 5.8, 4.3).
//
// A function returns None, having done nothing, for a call that is not ordinary: other types, strides, devices, a gradient
// asked for, an argument that the library refuses.  ops.py then goes the long way, which serves or refuses it.
//
// bind(handle, error, get_device, get_stream): the entry points of the library that _lib has loaded, its exception, and
// torch's current device and current raw stream of a device.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <dlfcn.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "camhip.h"

namespace {

PyObject *g_error = nullptr, *g_get_device = nullptr, *g_get_stream = nullptr;
decltype(&camhipGetLastErrorMsg) g_last_error = nullptr;
decltype(&camhipMoeRouteGroupedGetWorkspaceSize) g_get_route = nullptr;
decltype(&camhipAddRmsNormGetWorkspaceSize) g_get_norm = nullptr;
decltype(&camhipQuantMatmulGetWorkspaceSize) g_get_qmm = nullptr;
decltype(&camhipMoeDecodeLayerGetWorkspaceSize) g_get_layer = nullptr;
decltype(&camhipLoraAddGetWorkspaceSize) g_get_lora = nullptr;
decltype(&camhipReleaseExecutor) g_release = nullptr;
using RunFn = camhipStatus (*)(void *, uint64_t, camhipExecutor *, void *);
RunFn g_run_route = nullptr, g_run_norm = nullptr, g_run_qmm = nullptr, g_run_layer = nullptr, g_run_lora = nullptr;

// A tensor of a call: plain, on the GPU, without a gradient to be recorded.  nullptr: not ordinary.
const at::Tensor *plain(PyObject *o)
{
    if (!THPVariable_CheckExact(o))
        return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || (t.requires_grad() && c10::GradMode::is_enabled()))
        return nullptr;
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())  // (there is level 0 only)
        return nullptr;
    return &t;
}
// the same, absent for Python's None
bool optional(PyObject *o, const at::Tensor *&t)
{
    t = o == Py_None ? nullptr : plain(o);
    return t || o == Py_None;
}
bool vector_of(const at::Tensor &t, int64_t n) { return t.dim() == 1 && t.size(0) == n && t.is_contiguous(); }
bool is_fp32(const at::Tensor &t) { return t.scalar_type() == at::kFloat; }
// CAMHIP_DTYPE_*, -1 for none
int64_t code(at::ScalarType s)
{
    return s == at::kBFloat16 ? CAMHIP_DTYPE_BF16 : s == at::kHalf ? CAMHIP_DTYPE_FP16 : s == at::kFloat ? CAMHIP_DTYPE_FP32 : -1;
}
bool integer(PyObject *o, int64_t &v)
{
    if (!PyLong_CheckExact(o))
        return false;
    int over = 0;
    v = PyLong_AsLongLongAndOverflow(o, &over);
    return !over;
}
bool number(PyObject *o, double &v)
{
    if (!PyFloat_CheckExact(o))
        return false;
    v = PyFloat_AS_DOUBLE(o);
    return true;
}
bool is_string(PyObject *o, const char *s) { return PyUnicode_CheckExact(o) && PyUnicode_CompareWithASCIIString(o, s) == 0; }
// rows of contiguous elements, `step` elements apart
bool rows_of(const at::Tensor &t, int64_t &step)
{
    if (t.dim() != 2 || t.stride(1) != 1)
        return false;
    step = t.size(0) > 1 ? t.stride(0) : t.size(1);
    return step >= t.size(1);
}

// The current stream of the current device, which has to be where all of the tensors are.  1: yes, 0: not ordinary, -1: error.
int current_stream(std::initializer_list<const at::Tensor *> tensors, void *&stream)
{
    PyObject *d = PyObject_CallNoArgs(g_get_device);
    if (!d)
        return -1;
    const long index = PyLong_AsLong(d);
    for (const at::Tensor *t : tensors)
        if (t && t->get_device() != index) {
            Py_DECREF(d);
            return 0;
        }
    PyObject *s = PyObject_CallOneArg(g_get_stream, d);
    Py_DECREF(d);
    if (!s)
        return -1;
    stream = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    return PyErr_Occurred() ? -1 : 1;
}

bool launch(const char *name, RunFn run, camhipExecutor *ex, void *stream, void *workspace = nullptr, uint64_t bytes = 0)
{
    camhipStatus st;
    Py_BEGIN_ALLOW_THREADS
    st = run(workspace, bytes, ex, stream);
    Py_END_ALLOW_THREADS
    if (st != CAMHIP_SUCCESS)
        PyErr_Format(g_error, "%s failed (%d): %s", name, (int)st, g_last_error());
    return st == CAMHIP_SUCCESS;
}
// the same with a workspace, of torch's allocator
bool launch_ws(const char *name, RunFn run, camhipExecutor *ex, void *stream, uint64_t bytes, const at::Tensor &like)
{
    at::Tensor ws;
    try {
        ws = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    } catch (...) {
        g_release(ex);
        throw;
    }
    return launch(name, run, ex, stream, bytes ? ws.mutable_data_ptr() : nullptr, bytes);
}
PyObject *tuple_of(std::initializer_list<at::Tensor> tensors)
{
    PyObject *r = PyTuple_New((Py_ssize_t)tensors.size());
    Py_ssize_t i = 0;
    for (const at::Tensor &t : tensors) {
        PyObject *o = r ? THPVariable_Wrap(t) : nullptr;
        if (!o) {
            Py_XDECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

#define ORDINARY(cond)                                                                                               \
    do {                                                                                                             \
        if (!(cond))                                                                                                 \
            Py_RETURN_NONE;                                                                                          \
    } while (0)
#define STREAM(stream, ...)                                                                                          \
    void *stream = nullptr;                                                                                          \
    const int here = current_stream({__VA_ARGS__}, stream);                                                          \
    if (here < 0)                                                                                                    \
        return nullptr;                                                                                              \
    ORDINARY(here)

// logits, bias, topk, n_group, topk_group, score_func, group_score, renormalize, routed_scaling
PyObject *route_grouped(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    ORDINARY(n == 9 && g_error);
    const at::Tensor *lg = plain(a[0]), *bias = nullptr;
    int64_t K, G, KG, step;
    double scaling;
    ORDINARY(lg && optional(a[1], bias) && integer(a[2], K) && integer(a[3], G) && integer(a[4], KG) && number(a[8], scaling));
    ORDINARY(code(lg->scalar_type()) >= 0 && rows_of(*lg, step) && K > 0 && K <= 16 && PyBool_Check(a[7]));
    const int64_t T = lg->size(0), E = lg->size(1);
    ORDINARY(!bias || (is_fp32(*bias) && vector_of(*bias, E)));
    const bool softmax = is_string(a[5], "softmax"), top2 = is_string(a[6], "top2");
    ORDINARY((softmax || is_string(a[5], "sigmoid")) && (top2 || is_string(a[6], "max")));
    STREAM(stream, lg, bias);
    at::Tensor idx = at::empty({T, K}, lg->options().dtype(at::kInt)), w = at::empty({T, K}, lg->options().dtype(at::kFloat));
    uint64_t need = 0;
    camhipExecutor *ex = nullptr;
    ORDINARY(g_get_route(lg->const_data_ptr(), bias ? (const float *)bias->const_data_ptr() : nullptr, T, E, K,
                         code(lg->scalar_type()), step, G, KG, softmax ? CAMHIP_ROUTE_SOFTMAX : CAMHIP_ROUTE_SIGMOID,
                         top2 ? CAMHIP_ROUTE_GROUP_TOP2 : CAMHIP_ROUTE_GROUP_MAX, a[7] == Py_True, scaling,
                         (int32_t *)idx.mutable_data_ptr(), (float *)w.mutable_data_ptr(), nullptr, &need,
                         &ex) == CAMHIP_SUCCESS);
    return launch("camhipMoeRouteGrouped", g_run_route, ex, stream) ? tuple_of({idx, w}) : nullptr;
    END_HANDLE_TH_ERRORS
}

// x, residual, weight, eps, out_quant (0, 2, 3)
PyObject *add_rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    ORDINARY(n == 5 && g_error);
    const at::Tensor *x = plain(a[0]), *w = plain(a[2]), *res = nullptr;
    int64_t quant, step;
    double eps;
    ORDINARY(x && w && optional(a[1], res) && number(a[3], eps) && integer(a[4], quant));
    const at::ScalarType type = x->scalar_type();
    ORDINARY((type == at::kBFloat16 || type == at::kHalf) && rows_of(*x, step) && (quant == 0 || quant == 2 || quant == 3));
    const int64_t T = x->size(0), H = x->size(1);
    ORDINARY((w->scalar_type() == type || is_fp32(*w)) && vector_of(*w, H));
    ORDINARY(!res || (res->scalar_type() == type && res->dim() == 2 && res->size(0) == T && res->size(1) == H &&
                      res->is_contiguous()));
    STREAM(stream, x, w, res);
    const auto opt = x->options();
    at::Tensor y = at::empty({T, H}, quant == 0 ? opt : opt.dtype(quant == 2 ? at::kChar : at::kFloat8_e4m3fn));
    at::Tensor scale = quant == 3 ? at::empty_strided({T, H / 128}, {1, T}, opt.dtype(at::kFloat))
                                  : at::empty({quant == 2 ? T : 0}, opt.dtype(at::kFloat));
    at::Tensor added = res ? at::empty({T, H}, opt) : at::empty({0}, opt);
    uint64_t need = 0;
    camhipExecutor *ex = nullptr;
    ORDINARY(g_get_norm(x->const_data_ptr(), res ? res->const_data_ptr() : nullptr, w->const_data_ptr(), T, H, step, code(type),
                        code(w->scalar_type()), quant == 3 ? CAMHIP_QUANT_FP8_BLOCK_KMAJOR : quant, eps, y.mutable_data_ptr(),
                        (float *)scale.mutable_data_ptr(), added.mutable_data_ptr(), &need, &ex) == CAMHIP_SUCCESS);
    return launch("camhipAddRmsNorm", g_run_norm, ex, stream) ? tuple_of({y, scale, added}) : nullptr;
    END_HANDLE_TH_ERRORS
}

// x, x_scale, weight, weight_scale, bias, out_dtype
PyObject *quant_matmul(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    ORDINARY(n == 6 && g_error);
    const at::Tensor *x = plain(a[0]), *xs = plain(a[1]), *w = plain(a[2]), *ws = plain(a[3]), *bias = nullptr;
    ORDINARY(x && xs && w && ws && optional(a[4], bias) && (a[5] == Py_None || THPDtype_Check(a[5])));
    const at::ScalarType type = a[5] == Py_None ? at::kBFloat16 : reinterpret_cast<THPDtype *>(a[5])->scalar_type;
    ORDINARY(code(type) >= 0 && x->scalar_type() == at::kChar && w->scalar_type() == at::kChar && x->dim() == 2 &&
             w->dim() == 2 && x->is_contiguous() && w->is_contiguous() && x->size(1) == w->size(1));
    const int64_t M = x->size(0), N = w->size(0), K = x->size(1);
    ORDINARY(is_fp32(*xs) && vector_of(*xs, M) && is_fp32(*ws) && vector_of(*ws, N));
    ORDINARY(!bias || (is_fp32(*bias) && vector_of(*bias, N)));
    STREAM(stream, x, xs, w, ws, bias);
    at::Tensor out = at::empty({M, N}, x->options().dtype(type));
    uint64_t need = 0;
    camhipExecutor *ex = nullptr;
    ORDINARY(g_get_qmm(x->const_data_ptr(), (const float *)xs->const_data_ptr(), w->const_data_ptr(),
                       (const float *)ws->const_data_ptr(), bias ? (const float *)bias->const_data_ptr() : nullptr, M, N, K,
                       code(type), out.mutable_data_ptr(), &need, &ex) == CAMHIP_SUCCESS);
    return launch("camhipQuantMatmul", g_run_qmm, ex, stream) ? THPVariable_Wrap(out) : nullptr;
    END_HANDLE_TH_ERRORS
}

// a weight [lead..., n, k] with its scales: none (bf16), [lead..., n] (int8), [lead..., n / 128, k / 128] (fp8)
bool weight_of(const at::Tensor *w, const at::Tensor *s, at::ScalarType type, at::IntArrayRef shape)
{
    if (w->scalar_type() != type || w->sizes() != shape || !w->is_contiguous())
        return false;
    if (type == at::kBFloat16)
        return !s;
    if (!s || !is_fp32(*s) || !s->is_contiguous())
        return false;
    const size_t d = shape.size();
    if (type == at::kChar)
        return s->sizes() == shape.slice(0, d - 1);
    if (s->dim() != (int64_t)d)
        return false;
    for (size_t i = 0; i < d; ++i)
        if (s->size((int64_t)i) != (i + 2 < d ? shape[i] : shape[i] / 128))
            return false;
    return true;
}
template <typename T = void> T *ptr(const at::Tensor *t) { return t ? (T *)t->const_data_ptr() : nullptr; }

// x, router, bias, w1, s1, w2, s2, topk, n_group, topk_group, score_func, group_score, renormalize, routed_scaling, share w1, s1,
// w2, s2, active mask
PyObject *moe_decode_layer(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    ORDINARY(n == 19 && g_error);
    const at::Tensor *x = plain(a[0]), *router = plain(a[1]), *w1 = plain(a[3]), *w2 = plain(a[5]);
    const at::Tensor *bias, *s1, *s2, *sw1, *ss1, *sw2, *ss2, *mask;
    int64_t K, G, KG;
    double scaling;
    ORDINARY(x && router && w1 && w2 && optional(a[2], bias) && optional(a[4], s1) && optional(a[6], s2) && optional(a[14], sw1) &&
             optional(a[15], ss1) && optional(a[16], sw2) && optional(a[17], ss2) && optional(a[18], mask));
    ORDINARY(integer(a[7], K) && integer(a[8], G) && integer(a[9], KG) && PyBool_Check(a[12]) && number(a[13], scaling));
    const bool softmax = is_string(a[10], "softmax"), top2 = is_string(a[11], "top2");
    ORDINARY((softmax || is_string(a[10], "sigmoid")) && (top2 || is_string(a[11], "max")));
    ORDINARY(x->dim() == 2 && x->scalar_type() == at::kBFloat16 && x->is_contiguous() && w1->dim() == 3 && K > 0 && K <= 16);
    const int64_t T = x->size(0), H = x->size(1), E = w1->size(0), I = w1->size(1) / 2;
    const at::ScalarType type = w1->scalar_type();
    ORDINARY(T <= 16 && w1->size(1) % 2 == 0 && (type == at::kBFloat16 || type == at::kChar || type == at::kFloat8_e4m3fn));
    ORDINARY(router->dim() == 2 && router->size(0) == E && router->size(1) == H && router->is_contiguous() &&
             (is_fp32(*router) || router->scalar_type() == at::kBFloat16));
    ORDINARY(!bias || (is_fp32(*bias) && vector_of(*bias, E)));
    ORDINARY(!mask || (mask->scalar_type() == at::kBool && vector_of(*mask, T)));
    ORDINARY(weight_of(w1, s1, type, {E, 2 * I, H}) && weight_of(w2, s2, type, {E, H, I}));
    ORDINARY(!sw1 == !sw2 && (sw1 || (!ss1 && !ss2)));
    int64_t Is = 0;
    if (sw1) {
        ORDINARY(sw1->dim() == 2 && sw1->size(0) > 0 && sw1->size(0) % 2 == 0);
        Is = sw1->size(0) / 2;
        ORDINARY(weight_of(sw1, ss1, type, {2 * Is, H}) && weight_of(sw2, ss2, type, {H, Is}));
    }
    STREAM(stream, x, router, bias, w1, s1, w2, s2, sw1, ss1, sw2, ss2, mask);
    const auto opt = x->options();
    at::Tensor out = at::empty({T, H}, opt), idx = at::empty({T, K}, opt.dtype(at::kInt)), w = at::empty({T, K}, opt.dtype(at::kFloat));
    uint64_t need = 0;
    camhipExecutor *ex = nullptr;
    ORDINARY(g_get_layer(ptr<const uint16_t>(x), ptr(router), ptr<const float>(bias), ptr(w1), ptr<const float>(s1), ptr(w2),
                         ptr<const float>(s2), ptr(sw1), ptr<const float>(ss1), ptr(sw2), ptr<const float>(ss2),
                         ptr<const uint8_t>(mask), T, H, E, 2 * I, 2 * Is, K,
                         type == at::kBFloat16 ? CAMHIP_DTYPE_BF16 : type == at::kChar ? CAMHIP_DTYPE_INT8 : CAMHIP_DTYPE_FP8,
                         code(router->scalar_type()), G, KG, softmax ? CAMHIP_ROUTE_SOFTMAX : CAMHIP_ROUTE_SIGMOID,
                         top2 ? CAMHIP_ROUTE_GROUP_TOP2 : CAMHIP_ROUTE_GROUP_MAX, a[12] == Py_True, scaling,
                         (uint16_t *)out.mutable_data_ptr(), (int32_t *)idx.mutable_data_ptr(), (float *)w.mutable_data_ptr(), &need,
                         &ex) == CAMHIP_SUCCESS);
    return launch_ws("camhipMoeDecodeLayer", g_run_layer, ex, stream, need, *x) ? tuple_of({out, idx, w}) : nullptr;
    END_HANDLE_TH_ERRORS
}

// base, x, lora_a, lora_b, adapter_ids, scaling, x_scale, out_dtype
PyObject *lora_add(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    ORDINARY(n == 8 && g_error);
    const at::Tensor *base = plain(a[0]), *x = plain(a[1]), *la = plain(a[2]), *lb = plain(a[3]), *ids = plain(a[4]), *scaling, *xs;
    ORDINARY(base && x && la && lb && ids && optional(a[5], scaling) && optional(a[6], xs) && (a[7] == Py_None || THPDtype_Check(a[7])));
    int64_t bstep, xstep;
    ORDINARY(rows_of(*base, bstep) && rows_of(*x, xstep) && la->dim() == 3 && la->is_contiguous() && lb->is_contiguous());
    const int64_t m = x->size(0), k = x->size(1), nn = base->size(1), L = la->size(0), r = la->size(1);
    const at::ScalarType type = la->scalar_type(), bt = base->scalar_type();
    const bool int8 = x->scalar_type() == at::kChar;
    ORDINARY((type == at::kBFloat16 || type == at::kHalf) && (bt == at::kBFloat16 || bt == at::kHalf || bt == at::kFloat));
    ORDINARY(base->size(0) == m && la->size(2) == k && lb->scalar_type() == type && lb->sizes() == at::IntArrayRef({L, nn, r}));
    ORDINARY((int8 || x->scalar_type() == type) && int8 == (xs != nullptr) && (!xs || (is_fp32(*xs) && vector_of(*xs, m))));
    ORDINARY(ids->scalar_type() == at::kInt && vector_of(*ids, m) && (!scaling || (is_fp32(*scaling) && vector_of(*scaling, L))));
    const at::ScalarType ot = a[7] != Py_None ? reinterpret_cast<THPDtype *>(a[7])->scalar_type : bt == at::kFloat ? type : bt;
    ORDINARY(ot == at::kBFloat16 || ot == at::kHalf);
    STREAM(stream, base, x, la, lb, ids, scaling, xs);
    at::Tensor out = at::empty({m, nn}, base->options().dtype(ot));
    uint64_t need = 0;
    camhipExecutor *ex = nullptr;
    ORDINARY(g_get_lora(ptr(base), ptr(x), ptr<const float>(xs), ptr(la), ptr(lb), ptr<const int32_t>(ids), ptr<const float>(scaling), m, nn,
                        k, r, L, bstep, xstep, code(bt), int8 ? CAMHIP_DTYPE_INT8 : code(type), code(type), code(ot),
                        out.mutable_data_ptr(), &need, &ex) == CAMHIP_SUCCESS);
    return launch_ws("camhipLoraAdd", g_run_lora, ex, stream, need, *base) ? THPVariable_Wrap(out) : nullptr;
    END_HANDLE_TH_ERRORS
}

template <typename F> bool resolve(void *lib, const char *name, F &out)
{
    out = (F)dlsym(lib, name);
    if (!out)
        PyErr_Format(PyExc_ImportError, "the library has no %s", name);
    return out != nullptr;
}

PyObject *bind(PyObject *, PyObject *args)
{
    PyObject *handle, *type, *device, *stream;
    if (!PyArg_ParseTuple(args, "OOOO", &handle, &type, &device, &stream))
        return nullptr;
    void *lib = PyLong_AsVoidPtr(handle);
    if (PyErr_Occurred())
        return nullptr;
    if (!resolve(lib, "camhipMoeRouteGroupedGetWorkspaceSize", g_get_route) ||
        !resolve(lib, "camhipMoeRouteGrouped", g_run_route) ||
        !resolve(lib, "camhipAddRmsNormGetWorkspaceSize", g_get_norm) || !resolve(lib, "camhipAddRmsNorm", g_run_norm) ||
        !resolve(lib, "camhipQuantMatmulGetWorkspaceSize", g_get_qmm) || !resolve(lib, "camhipQuantMatmul", g_run_qmm) ||
        !resolve(lib, "camhipMoeDecodeLayerGetWorkspaceSize", g_get_layer) || !resolve(lib, "camhipMoeDecodeLayer", g_run_layer) ||
        !resolve(lib, "camhipLoraAddGetWorkspaceSize", g_get_lora) || !resolve(lib, "camhipLoraAdd", g_run_lora) ||
        !resolve(lib, "camhipReleaseExecutor", g_release) || !resolve(lib, "camhipGetLastErrorMsg", g_last_error))
        return nullptr;
    Py_INCREF(device);
    Py_XSETREF(g_get_device, device);
    Py_INCREF(stream);
    Py_XSETREF(g_get_stream, stream);
    Py_INCREF(type);
    Py_XSETREF(g_error, type);
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD(route_grouped), METHOD(add_rms_norm), METHOD(quant_matmul), METHOD(moe_decode_layer), METHOD(lora_add),
                           {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_camops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__camops(void) { return PyModule_Create(&g_module); }
