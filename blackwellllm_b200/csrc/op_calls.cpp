// The way from Python to the kernels of the 8-bit cache and of the log probabilities: operands looked over, outputs allocated on the current
// stream, the kernel's entry point called.  As Python these steps took 8 of a small call's 13 us (an output's allocation alone 2.4, a call
// with twenty numbers through ctypes 1.5); what is left is mostly the launch itself.
//
// An entry point comes as its address (kernels/ops.py has the libraries).  A call returns its outputs, or the entry point's error code as a
// number, or None where the operands do not fit: what is wrong with them is for the caller to say.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

namespace {

using ll = long long;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool is(const at::Tensor* t, at::ScalarType type, int device) {
    return t && t->is_cuda() && t->get_device() == device && t->scalar_type() == type && t->is_contiguous();
}
bool small(int64_t n) { return n >= 0 && n <= 0x7fffffff; }
// A Python number that fits an int.
bool whole(PyObject* o, int& n) {
    int over = 0;
    const ll v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over || (v == -1 && PyErr_Occurred())) { PyErr_Clear(); return false; }
    if (v < -0x80000000ll || v > 0x7fffffffll) return false;
    n = (int)v;
    return true;
}
template <typename F> F entry(PyObject* address) { return reinterpret_cast<F>(PyLong_AsVoidPtr(address)); }
// (past the dispatcher, which takes as long as the allocation)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, int device) {
    return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}
void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }
const float* floats(const at::Tensor* t) { return t ? (const float*)t->const_data_ptr() : nullptr; }
const int* ints(const at::Tensor* t) { return (const int*)t->const_data_ptr(); }

// Pages [num_pages, nkv, page_size, hd], their scales and the table of blocks, all on the current device.
struct Pages {
    const at::Tensor *k, *v, *ks, *vs, *table;
    int device, num_pages, nkv, page_size, hd;
    bool take(PyObject* const* a) {
        k = tensor(a[0]); v = tensor(a[1]); ks = tensor(a[2]); vs = tensor(a[3]); table = tensor(a[4]);
        device = c10::cuda::current_device();
        if (!is(k, at::kChar, device) || !is(v, at::kChar, device) || !is(ks, at::kFloat, device) || !is(vs, at::kFloat, device) ||
            !is(table, at::kInt, device))
            return false;
        const auto s = k->sizes();
        if (s.size() != 4 || v->sizes() != s || ks->sizes() != s.slice(0, 3) || vs->sizes() != s.slice(0, 3) || table->dim() != 2) return false;
        for (int64_t n : s) if (!small(n)) return false;
        num_pages = (int)s[0]; nkv = (int)s[1]; page_size = (int)s[2]; hd = (int)s[3];
        return hd > 0 && hd % 16 == 0 && hd <= 256 && small(table->size(0)) && small(table->size(1));
    }
};

using AppendFn = int (*)(const void*, int, int, ll, const float*, int, int, void*, int, void*, void*, float*, float*, const int*, const int*,
                         const int*, int, int, int, int, int, int, int, int, void*);
// (entry, k, v, k_scale, v_scale, table, qkv, positions, req_of_token, nh, turns or None, paired, append)
PyObject* quant_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Pages p;
    int nh;
    if (n != 13 || !p.take(a + 1) || !whole(a[9], nh)) Py_RETURN_NONE;
    const at::Tensor *qkv = tensor(a[6]), *pos = tensor(a[7]), *req = tensor(a[8]), *turns = a[10] == Py_None ? nullptr : tensor(a[10]);
    if (!qkv || !qkv->is_cuda() || qkv->get_device() != p.device || !is(pos, at::kInt, p.device) || !is(req, at::kInt, p.device)) Py_RETURN_NONE;
    const bool wide = qkv->scalar_type() == at::kFloat;
    const int64_t d = qkv->dim();
    if ((!wide && qkv->scalar_type() != at::kBFloat16) || (d == 3 ? !wide || qkv->size(0) < 1 : d != 2)) Py_RETURN_NONE;
    const int64_t T = qkv->size(d - 2), W = qkv->size(d - 1), planes = d == 3 ? qkv->size(0) : 1;
    if (!small(T) || !small(planes) || nh < 0 || W != ((int64_t)nh + 2 * (int64_t)p.nkv) * p.hd || pos->numel() != T || req->numel() != T) Py_RETURN_NONE;
    if (d == 3 ? T > 0 && (qkv->stride(2) != 1 || (T > 1 && qkv->stride(1) != W)) : !qkv->is_contiguous()) Py_RETURN_NONE;
    int64_t rd = 0;
    if (a[10] != Py_None) {
        if (!is(turns, at::kFloat, p.device) || turns->dim() != 2 || turns->size(0) != T || turns->size(1) % 2 || turns->size(1) > p.hd) Py_RETURN_NONE;
        rd = turns->size(1);
    }
    const int paired = PyObject_IsTrue(a[11]), append = PyObject_IsTrue(a[12]);
    if (paired < 0 || append < 0) return nullptr;
    at::Tensor q = fresh({T, (int64_t)nh * p.hd}, at::kBFloat16, p.device);
    if (T > 0) {
        const int code = entry<AppendFn>(a[0])(qkv->const_data_ptr(), wide ? 0 : 1, (int)planes, d == 3 ? qkv->stride(0) : 0, rd ? floats(turns) : nullptr, (int)rd,
                                               paired, q.mutable_data_ptr(), nh, p.k->data_ptr(), p.v->data_ptr(), (float*)p.ks->data_ptr(),
                                               (float*)p.vs->data_ptr(), ints(pos), ints(req), ints(p.table), (int)T, (int)p.table->size(0),
                                               (int)p.table->size(1), p.page_size, p.num_pages, p.nkv, p.hd, append, stream());
        if (code) return PyLong_FromLong(code);
    }
    return THPVariable_Wrap(std::move(q));
    END_HANDLE_TH_ERRORS
}

using ReadFn = int (*)(const void*, const void*, const float*, const float*, const int*, const int*, const int*, void*, void*, int, int, int, int,
                       int, int, int, int, void*);
PyObject* pair(at::Tensor&& x, at::Tensor&& y) {
    PyObject* t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(x)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(y)));
    return t;
}
// (entry, k, v, k_scale, v_scale, table, positions, req_of_token, whether the outputs are float32 (else bfloat16))
PyObject* quant_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Pages p;
    if (n != 9 || !p.take(a + 1)) Py_RETURN_NONE;
    const at::Tensor *pos = tensor(a[6]), *req = tensor(a[7]);
    if (!is(pos, at::kInt, p.device) || !is(req, at::kInt, p.device) || pos->numel() != req->numel() || !small(pos->numel())) Py_RETURN_NONE;
    const bool wide = a[8] == Py_True;
    const int64_t T = pos->numel();
    const at::ScalarType type = wide ? at::kFloat : at::kBFloat16;
    at::Tensor k = fresh({T, p.nkv, p.hd}, type, p.device), v = fresh({T, p.nkv, p.hd}, type, p.device);
    if (T > 0) {
        const int code = entry<ReadFn>(a[0])(p.k->const_data_ptr(), p.v->const_data_ptr(), floats(p.ks), floats(p.vs), ints(pos), ints(req), ints(p.table),
                                             k.mutable_data_ptr(), v.mutable_data_ptr(), wide ? 0 : 1, (int)T, (int)p.table->size(0), (int)p.table->size(1),
                                             p.page_size, p.num_pages, p.nkv, p.hd, stream());
        if (code) return PyLong_FromLong(code);
    }
    return pair(std::move(k), std::move(v));
    END_HANDLE_TH_ERRORS
}

using FewFn = int (*)(const void*, const void*, const void*, const float*, const float*, void*, const int*, const int*, const int*, const int*, int,
                      const int*, const int*, int, int, int, int, int, int, int, int, float, const float*, float*, ll, ll*, int*, void*);
using RoomFn = ll (*)(const int*, const int*, int, int, int, int, int, int);
using ManyFn = int (*)(const void*, const void*, const void*, const float*, const float*, void*, const int*, const int*, int, const int*, const int*,
                       int, int, int, int, int, int, int, int, float, const float*, float*, ll, void*);
constexpr int ERR_ROOM = -11;
// A list's or tuple's first n numbers, each a length or a position.
bool numbers(PyObject* list, int n, std::vector<int>& out) {
    if (!(PyList_Check(list) || PyTuple_Check(list)) || PySequence_Fast_GET_SIZE(list) < n) return false;
    PyObject** items = PySequence_Fast_ITEMS(list);
    out.resize(n);
    for (int i = 0; i < n; ++i) if (!whole(items[i], out[i])) return false;
    return true;
}
// (few rows' entry, many rows' room, many rows' entry, k, v, k_scale, v_scale, table, q, cu_q, q_start, kv_len, lengths, starts, T, R, nh, most query
// heads a kv head, most rows of few, scale, window, chunk, bound, sink or None, a captured step's division or None) -> (out, entry points called)
PyObject* quant_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Pages p;
    int T, R, nh, most_group, few_rows, window, chunk, bound;
    if (n != 25 || !p.take(a + 3) || !whole(a[14], T) || !whole(a[15], R) || !whole(a[16], nh) || !whole(a[17], most_group) || !whole(a[18], few_rows) ||
        !whole(a[20], window) || !whole(a[21], chunk) || !whole(a[22], bound))
        Py_RETURN_NONE;
    const at::Tensor *q = tensor(a[8]), *cu = tensor(a[9]), *start = tensor(a[10]), *len = tensor(a[11]), *sink = nullptr, *dealt = nullptr;
    if (!is(q, at::kBFloat16, p.device) || !is(cu, at::kInt, p.device) || !is(start, at::kInt, p.device) || !is(len, at::kInt, p.device)) Py_RETURN_NONE;
    if (p.nkv < 1 || nh < 1 || nh % p.nkv || nh / p.nkv > most_group || q->dim() != 2 || q->size(0) != T || q->size(1) != (int64_t)nh * p.hd) Py_RETURN_NONE;
    if (T < 0 || R < 0 || p.table->size(0) < R || cu->numel() < (int64_t)R + 1 || start->numel() < R || len->numel() < R) Py_RETURN_NONE;
    if (a[23] != Py_None && (!is(sink = tensor(a[23]), at::kFloat, p.device) || sink->numel() != nh)) Py_RETURN_NONE;
    if (a[24] != Py_None && !is(dealt = tensor(a[24]), at::kInt, p.device)) Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(a[19]);
    if (PyErr_Occurred()) return nullptr;
    std::vector<int> lens, starts;
    if (!(scale > 0.0) || !numbers(a[12], R, lens) || !numbers(a[13], R, starts)) Py_RETURN_NONE;
    ll sum = 0, most = 0;
    int least = 0x7fffffff;
    for (int i : lens) { sum += i; most = i > most ? i : most; least = i < least ? i : least; }
    if (sum != T) Py_RETURN_NONE;
    const int G = nh / p.nkv, blocks = (int)p.table->size(1);
    at::Tensor out = fresh(q->sizes(), at::kBFloat16, p.device);
    long calls = 0;
    if (T > 0) {
        if (most * G > few_rows) {
            const ll need = entry<RoomFn>(a[1])(lens.data(), starts.data(), R, few_rows, G, p.nkv, window, chunk);
            if (need < 0) return PyLong_FromLongLong(need);
            at::Tensor room = fresh({(int64_t)need}, at::kFloat, p.device);
            const int code = entry<ManyFn>(a[2])(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(), floats(p.ks), floats(p.vs),
                                                 out.mutable_data_ptr(), ints(len), ints(p.table), blocks, lens.data(), starts.data(), R, few_rows, nh, p.nkv,
                                                 p.page_size, p.num_pages, window, chunk, (float)scale, floats(sink), (float*)room.mutable_data_ptr(), need,
                                                 stream());
            if (code) return PyLong_FromLong(code);
            ++calls;
        }
        if ((ll)least * G <= few_rows) {
            // many slices of few requests join through memory, and a captured step's are divided there: the entry point says how much it takes
            at::Tensor room;
            ll have = 0, need = 0;
            int code;
            do {
                if (need) { room = fresh({(int64_t)need}, at::kFloat, p.device); have = need; }
                code = entry<FewFn>(a[0])(q->const_data_ptr(), p.k->const_data_ptr(), p.v->const_data_ptr(), floats(p.ks), floats(p.vs), out.mutable_data_ptr(),
                                          ints(cu), ints(start), ints(len), ints(p.table), blocks, lens.data(), starts.data(), R, nh, p.nkv, p.page_size,
                                          p.num_pages, window, chunk, bound, (float)scale, floats(sink), have ? (float*)room.mutable_data_ptr() : nullptr, have,
                                          &need, dealt ? (int*)dealt->data_ptr() : nullptr, stream());
            } while (code == ERR_ROOM && !have);
            if (code) return PyLong_FromLong(code);
            ++calls;
        }
    }
    PyObject* t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(t, 1, PyLong_FromLong(calls));
    return t;
    END_HANDLE_TH_ERRORS
}

using ProbsFn = int (*)(const float*, const int*, float*, float*, int*, int*, float*, int, int, int, ll, void*);
// (entry, logits, target, top, most of top) -> (log_prob, entropy, rank, top_ids, top_log_probs)
PyObject* token_log_probs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int top, most;
    if (n != 5 || !whole(a[3], top) || !whole(a[4], most)) Py_RETURN_NONE;
    const at::Tensor *x = tensor(a[1]), *target = tensor(a[2]);
    const int device = c10::cuda::current_device();
    if (!x || !x->is_cuda() || x->get_device() != device || x->scalar_type() != at::kFloat || x->dim() != 2 || !is(target, at::kInt, device)) Py_RETURN_NONE;
    const int64_t R = x->size(0), V = x->size(1);
    if (V < 1 || !small(R) || !small(V) || x->stride(1) != 1 || (R > 1 && x->stride(0) < V) || target->numel() != R || top < 0 || top > most || top > V)
        Py_RETURN_NONE;
    at::Tensor got[5] = {fresh({R}, at::kFloat, device), fresh({R}, at::kFloat, device), fresh({R}, at::kInt, device), fresh({R, top}, at::kInt, device),
                         fresh({R, top}, at::kFloat, device)};
    if (R > 0) {
        const int code = entry<ProbsFn>(a[0])(floats(x), ints(target), (float*)got[0].mutable_data_ptr(), (float*)got[1].mutable_data_ptr(),
                                              (int*)got[2].mutable_data_ptr(), (int*)got[3].mutable_data_ptr(), (float*)got[4].mutable_data_ptr(), (int)R, (int)V,
                                              top, R > 1 ? x->stride(0) : V, stream());
        if (code) return PyLong_FromLong(code);
    }
    PyObject* t = PyTuple_New(5);
    if (!t) return nullptr;
    for (int j = 0; j < 5; ++j) PyTuple_SET_ITEM(t, j, THPVariable_Wrap(std::move(got[j])));
    return t;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"quant_append", (PyCFunction)(void (*)(void))quant_append, METH_FASTCALL, nullptr},
                         {"quant_read", (PyCFunction)(void (*)(void))quant_read, METH_FASTCALL, nullptr},
                         {"quant_attention", (PyCFunction)(void (*)(void))quant_attention, METH_FASTCALL, nullptr},
                         {"token_log_probs", (PyCFunction)(void (*)(void))token_log_probs, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "op_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_op_calls() { return PyModule_Create(&module); }
