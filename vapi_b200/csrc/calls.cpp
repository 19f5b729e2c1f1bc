// The calls that a step of a few tokens makes most often, from Python's arguments to the launch in one piece: checks, outputs and the
// call of the kernel's C function.  Such a step (a prompt of a line: 65 products, 97 launches) is bound by what its launches cost the
// host, and of a product's 14 us there only about 3 are the launch; checking its operands one by one in Python, allocating its
// outputs through the Python binding and converting two dozen arguments through ctypes are the rest.
//
// A function here answers NotImplemented for anything but what the kernels take as it is (other types, layouts, devices or
// tensor classes): its caller in ops then goes through the same steps in Python, which name what is wrong.  A negative number is the C
// function's error code.  Once the C function has been called there is no way back to Python's steps, which would add to the stream, or move
// a state on, a second time: what goes wrong from there on is an error.  The C functions are given by address, so this library is linked
// with none of the kernels' ones.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

namespace {

struct Bad {};                              // not for this file: NotImplemented

const at::Tensor* tensor(PyObject* o) {     // None: null
    if (o == Py_None) return nullptr;
    if (!THPVariable_CheckExact(o)) throw Bad{};
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg()) throw Bad{};
    return &t;
}
const at::Tensor& need(PyObject* o, at::ScalarType type, int64_t dim) {
    const at::Tensor* t = tensor(o);
    if (!t || t->scalar_type() != type || t->dim() != dim || !t->is_contiguous()) throw Bad{};
    return *t;
}
// a vector of floats, as many as the kernel reads or more (`most`: no more than that), or none
const float* floats(PyObject* o, int64_t least, int64_t most = INT64_MAX) {
    const at::Tensor* t = tensor(o);
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() < least || t->numel() > most) throw Bad{};
    return static_cast<const float*>(t->data_ptr());
}
const int* ints(PyObject* o, int64_t least) {
    const at::Tensor* t = tensor(o);
    if (!t || t->scalar_type() != at::kInt || !t->is_contiguous() || t->numel() < least) throw Bad{};
    return static_cast<const int*>(t->data_ptr());
}
void* address(PyObject* o) {                // None: null
    if (o == Py_None) return nullptr;
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) { PyErr_Clear(); throw Bad{}; }
    return p;
}
int integer(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if ((v == -1 && PyErr_Occurred()) || v > 0x7fffffffL || v < -0x7fffffffL) { PyErr_Clear(); throw Bad{}; }
    return (int)v;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); throw Bad{}; }
    return (float)v;
}
int size32(int64_t v) {
    if (v > 0x7fffffffLL) throw Bad{};
    return (int)v;
}
PyObject* wrap(const at::Tensor& t) {       // (null: a Python error)
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// The interpreter's lock is given up while one of these lives, and taken again however its block is left.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// body(called): sets `called` before it calls the C function
template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& body) {
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments instead of %zd", given, wanted);
        return nullptr;
    }
    bool called = false;
    const char* what = "an unknown exception";
    std::string text;
    try {
        return body(called);
    } catch (const Bad&) {
    } catch (const std::exception& e) {     // (what torch objects to, the same calls in Python say)
        text = e.what();
        what = text.c_str();
    } catch (...) {
    }
    if (called) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "a kernel's launch ended with an exception: %s", what);
        return nullptr;
    }
    PyErr_Clear();
    Py_RETURN_NOTIMPLEMENTED;
}

typedef int (*PlanFn)(int, int, int, int, int*, int*, int*);
typedef int (*ProductFn)(const void*, int, int, int, int, const void*, const float*, int, float, int, void*, float*, long long, const float*,
                         float*, float*, const float*, void*, int*, void*, const float*, int);
enum { EPI_BF16 = 0, EPI_SWIGLU = 1, EPI_RESID = 2, EPI_F32 = 3 };

// product(fn, plan, which of the plan's answers is the partial sums of squares, weight, act, xw, ss_in, eps, epilogue, bias, resid,
//         next_weight, status, xielu, glu, stream): ops._fused_product
PyObject* product(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 16, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<ProductFn>(address(a[0]));
        const auto plan = reinterpret_cast<PlanFn>(address(a[1]));
        const int answer = integer(a[2]), epi = integer(a[8]);
        if (!fn || !plan || answer < 0 || answer > 2 || epi < EPI_BF16 || epi > EPI_F32) throw Bad{};
        const at::Tensor& w = need(a[3], at::kBFloat16, 2);
        const bool norm = a[4] == Py_None;
        const at::Tensor& x = need(norm ? a[5] : a[4], at::kBFloat16, 2);
        const int N = size32(w.size(0)), K = size32(w.size(1)), M = size32(x.size(0));
        if (x.size(1) != K) throw Bad{};
        const float* ss = nullptr;
        int parts_in = 0;
        if (norm) {
            const at::Tensor& s = need(a[6], at::kFloat, 2);
            if (s.size(1) != M) throw Bad{};
            ss = static_cast<const float*>(s.data_ptr());
            parts_in = size32(s.size(0));
        } else if (a[6] != Py_None) {
            throw Bad{};
        }
        const float* bias = floats(a[9], N, N);
        const float* next_w = floats(a[11], N);
        const float* xielu = floats(a[13], 2);
        float* resid = nullptr;
        at::Tensor out, sums, weighted;
        const auto options = w.options();
        long long stride = N;
        if (epi == EPI_RESID) {
            const at::Tensor& r = need(a[10], at::kFloat, 2);
            if (r.size(0) != M || r.size(1) != N) throw Bad{};
            resid = static_cast<float*>(r.data_ptr());
            if (next_w) {
                int o[3] = {0, 0, 0};
                plan(N, K, M, epi, &o[0], &o[1], &o[2]);
                sums = at::empty({o[answer], M}, options.dtype(at::kFloat));
                weighted = at::empty({M, N}, options);
            }
        } else {
            if (a[10] != Py_None) throw Bad{};
            if (epi == EPI_SWIGLU) stride = N / 2;
            out = at::empty({M, stride}, epi == EPI_F32 ? options.dtype(at::kFloat) : options);
        }
        void* o = out.defined() ? out.data_ptr() : nullptr;
        float* so = sums.defined() ? static_cast<float*>(sums.data_ptr()) : nullptr;
        void* wo = weighted.defined() ? weighted.data_ptr() : nullptr;
        const float eps = real(a[7]);
        int* status = static_cast<int*>(address(a[12]));
        void* stream = address(a[15]);
        const int glu = integer(a[14]);
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(w.data_ptr(), N, K, M, norm ? 1 : 0, x.data_ptr(), ss, parts_in, eps, epi, epi == EPI_F32 ? nullptr : o,
                    epi == EPI_F32 ? static_cast<float*>(o) : nullptr, stride, bias, resid, so, next_w, wo, status, stream, xielu, glu);
        }
        if (rc != 0) return PyLong_FromLong(rc);
        if (epi != EPI_RESID) return wrap(out);
        PyObject* first = wrap(sums);
        PyObject* second = first ? wrap(weighted) : nullptr;
        PyObject* pair = second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return pair;
    });
}

typedef int (*ShortconvFn)(const void*, int, const float*, const float*, const float*, void*, long long, const int*, const int*, const int*,
                           const int*, void*, int, int, int, int, int, int*, void*);

// shortconv(fn, h3, in_bias, taps, conv_bias, state, state_slots, tok_seq, cu_q, positions, status, stream): ops.shortconv in bfloat16
PyObject* shortconv(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 12, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<ShortconvFn>(address(a[0]));
        const at::Tensor& h3 = need(a[1], at::kBFloat16, 2);
        const at::Tensor& taps = need(a[3], at::kFloat, 2);
        const int n = size32(h3.size(0)), H = size32(h3.size(1) / 3), L = size32(taps.size(0));
        if (!fn || h3.size(1) != 3LL * H || taps.size(1) != H) throw Bad{};
        const at::Tensor* state = tensor(a[5]);
        long long slot_stride = 0;
        int slots = 0;
        if (L > 1) {
            if (!state || state->scalar_type() != at::kBFloat16 || state->dim() != 3 || state->size(1) != L - 1 || state->size(2) != H ||
                state->stride(2) != 1 || state->stride(1) != H) throw Bad{};
            slot_stride = state->stride(0);
            slots = size32(state->size(0));
        }
        const at::Tensor* cu = tensor(a[8]);
        if (!cu || cu->scalar_type() != at::kInt || !cu->is_contiguous()) throw Bad{};
        const int seqs = size32(cu->numel() - 1);
        const float *in_bias = floats(a[2], 3LL * H), *conv_bias = floats(a[4], H);
        const int *state_slots = ints(a[6], seqs), *tok_seq = ints(a[7], n), *positions = ints(a[9], n);
        int* status = static_cast<int*>(address(a[10]));
        void* stream = address(a[11]);
        at::Tensor out = at::empty({n, H}, h3.options());
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(h3.data_ptr(), 1, in_bias, static_cast<const float*>(taps.data_ptr()), conv_bias, L > 1 ? state->data_ptr() : nullptr,
                    slot_stride, state_slots, tok_seq, static_cast<const int*>(cu->data_ptr()), positions, out.data_ptr(), n, seqs, H, L,
                    slots, status, stream);
        }
        return rc != 0 ? PyLong_FromLong(rc) : wrap(out);
    });
}

// ---- operators of serving in fewer bits ---------------------------------------------------------------
// (`device`: the current one; all of a call's tensors are on it, or Python's steps say which is not)
const at::Tensor& on(const at::Tensor& t, int device) {
    if (t.get_device() != device) throw Bad{};
    return t;
}
const at::Tensor* on(const at::Tensor* t, int device) {
    if (t) on(*t, device);
    return t;
}
const float* floats_on(PyObject* o, int64_t size, int device) {
    on(tensor(o), device);
    return floats(o, size, size);
}
const int* ints_on(PyObject* o, int64_t least, int device) {
    on(tensor(o), device);
    const int* p = ints(o, least);
    if (!p) throw Bad{};
    return p;
}
int type_code(const at::Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return 1;
    if (t.scalar_type() != at::kFloat) throw Bad{};
    return 0;
}
struct Codes { const at::Tensor* codes; const at::Tensor* exps; int pages, nkv, page_size, d; };
Codes cache8(PyObject* codes, PyObject* exps, int device) {
    const at::Tensor& c = on(need(codes, at::kFloat8_e4m3fn, 5), device);
    const at::Tensor& e = on(need(exps, at::kChar, 4), device);
    if (c.size(1) != 2 || c.size(0) == 0 || c.size(3) == 0 || c.size(3) % 16 != 0 || e.size(0) != c.size(0) || e.size(1) != 2 || e.size(2) != c.size(2) ||
        e.size(3) != c.size(3) / 16) throw Bad{};
    return {&c, &e, size32(c.size(0)), size32(c.size(2)), size32(c.size(3)), size32(c.size(4))};
}

typedef int (*Write8Fn)(const void*, int, const float*, const float*, float, const float*, const float*, int, void*, void*, void*, const int*, int, int,
                        int, int, int, int, int*, void*);

// write8(fn, qkv, nh, nkv, d, q_weight, k_weight, eps, cos, sin, rot, codes, exps, slots, status, stream, device): ops.qk_norm_rope_write8
PyObject* write8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 17, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<Write8Fn>(address(a[0]));
        const int nh = integer(a[2]), nkv = integer(a[3]), d = integer(a[4]), rot = integer(a[10]), device = integer(a[16]);
        const at::Tensor* x = on(tensor(a[1]), device);
        if (!fn || !x || x->dim() != 2 || !x->is_contiguous() || nh <= 0 || nkv <= 0 || d <= 0 || x->size(1) != (nh + 2LL * nkv) * d) throw Bad{};
        const int n = size32(x->size(0)), type = type_code(*x);
        const Codes c = cache8(a[11], a[12], device);
        if (c.nkv != nkv || c.d != d) throw Bad{};
        const at::Tensor *cs = on(tensor(a[8]), device), *sn = on(tensor(a[9]), device);
        if ((cs == nullptr) != (sn == nullptr)) throw Bad{};
        for (const at::Tensor* t : {cs, sn})
            if (t && (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != n || t->size(1) != rot / 2 || !t->is_contiguous())) throw Bad{};
        const float *qw = floats_on(a[5], d, device), *kw = floats_on(a[6], d, device);
        const int* slots = ints_on(a[13], n, device);
        const float eps = real(a[7]);
        int* status = static_cast<int*>(address(a[14]));
        void* stream = address(a[15]);
        at::Tensor q = at::empty({n, (int64_t)nh * d}, x->options());
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(x->data_ptr(), type, qw, kw, eps, cs ? static_cast<const float*>(cs->data_ptr()) : nullptr,
                    sn ? static_cast<const float*>(sn->data_ptr()) : nullptr, rot, q.data_ptr(), c.codes->data_ptr(), c.exps->data_ptr(), slots, n, nh, nkv, d,
                    c.page_size, c.pages, status, stream);
        }
        return rc != 0 ? PyLong_FromLong(rc) : wrap(q);
    });
}

typedef int (*Read8Fn)(const void*, const void*, const int*, void*, int, int, int, int, int, int, int*, void*);

// read8(fn, codes, exps, pages, float32 or not, status, stream, device): ops.cache8_read
PyObject* read8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<Read8Fn>(address(a[0]));
        const int f32 = integer(a[4]), device = integer(a[7]);
        const Codes c = cache8(a[1], a[2], device);
        const int* pages = ints_on(a[3], 0, device);
        const int count = size32(tensor(a[3])->numel());
        int* status = static_cast<int*>(address(a[5]));
        void* stream = address(a[6]);
        if (!fn) throw Bad{};
        at::Tensor out = at::empty({count, 2, c.nkv, c.page_size, c.d}, c.codes->options().dtype(f32 ? at::kFloat : at::kBFloat16));
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(c.codes->data_ptr(), c.exps->data_ptr(), pages, out.data_ptr(), f32 ? 0 : 1, count, c.nkv, c.d, c.page_size, c.pages, status, stream);
        }
        return rc != 0 ? PyLong_FromLong(rc) : wrap(out);
    });
}

typedef int (*Attention8Fn)(const void*, long long, const void*, const void*, int, const int*, int, const int*, const int*, void*, int, int, int, int, int,
                            int, int, int, int, float, int, int, int, int, int*, void*);

// attention8(fn, q, q_row_stride, codes, exps, block_table, cu_q, seqlens_k, n, num_seqs, max_q, max_k, nh, nkv, d, scale, window, splits, impl, settled,
//            status, stream, device): ops.paged_attention8
PyObject* attention8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 23, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<Attention8Fn>(address(a[0]));
        const int device = integer(a[22]), n = integer(a[8]), seqs = integer(a[9]), max_q = integer(a[10]), max_k = integer(a[11]);
        const int nh = integer(a[12]), nkv = integer(a[13]), d = integer(a[14]);
        const int64_t stride = integer(a[2]);
        const at::Tensor* q = on(tensor(a[1]), device);
        if (!fn || !q || q->dim() < 1 || q->stride(-1) != 1 || n < 0 || seqs < 0 || nh <= 0 || nkv <= 0 || nh % nkv != 0 || d <= 0 || stride < (int64_t)nh * d) throw Bad{};
        const int type = type_code(*q);
        if (n > 0 && (int64_t)q->storage().nbytes() < (q->storage_offset() + (n - 1) * stride + (int64_t)nh * d) * (int64_t)q->element_size()) throw Bad{};
        const Codes c = cache8(a[3], a[4], device);
        if (c.nkv != nkv || c.d != d) throw Bad{};
        const at::Tensor* table = on(tensor(a[5]), device);
        if (!table || table->scalar_type() != at::kInt || table->dim() != 2 || table->stride(1) != 1 || table->size(0) < seqs) throw Bad{};
        const int *cu = ints_on(a[6], seqs + 1LL, device), *kl = ints_on(a[7], seqs, device);
        const float scale = real(a[15]);
        const int window = integer(a[16]), splits = integer(a[17]), impl = integer(a[18]), settled = integer(a[19]), table_stride = size32(table->stride(0));
        int* status = static_cast<int*>(address(a[20]));
        void* stream = address(a[21]);
        at::Tensor out = at::empty({n, (int64_t)nh * d}, q->options());
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(q->data_ptr(), stride, c.codes->data_ptr(), c.exps->data_ptr(), type, static_cast<const int*>(table->data_ptr()), table_stride, cu, kl,
                    out.data_ptr(), n, seqs, max_q, max_k, nh, nkv, d, c.page_size, c.pages, scale, window, splits, impl, settled, status, stream);
        }
        return rc != 0 ? PyLong_FromLong(rc) : wrap(out);
    });
}

typedef int (*Int4Fn)(const void*, const void*, int, int, int, const void*, int, const float*, void*, float*, int, int, int, void*);

// int4(fn, codes, scales, n, k, group, x, bias, gated, act, float32 or not, stream, device): ops.int4_linear and int4_linear_swiglu of few rows.
// (codes and scales are an Int4Weight's, laid out and checked by int4_pack)
PyObject* int4(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 13, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<Int4Fn>(address(a[0]));
        const int n = integer(a[3]), k = integer(a[4]), group = integer(a[5]), gated = integer(a[8]), act = integer(a[9]), f32 = integer(a[10]), device = integer(a[12]);
        const at::Tensor& codes = on(need(a[1], at::kInt, 4), device);
        const at::Tensor& scales = on(need(a[2], at::kInt, 4), device);
        const at::Tensor& x = on(need(a[6], at::kBFloat16, 2), device);
        if (!fn || x.size(1) != k || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) != 0 || (gated && (f32 || a[7] != Py_None))) throw Bad{};
        const int64_t tiles = (n + 15LL) / 16;
        if (n <= 0 || k <= 0 || group <= 0 || codes.numel() != tiles * ((k + 63LL) / 64) * 128 || scales.numel() != tiles * (group == 32 ? (k + 63LL) / 64 * 2 : k / group) * 16) throw Bad{};
        const int rows = size32(x.size(0));
        const float* bias = floats_on(a[7], n, device);
        void* stream = address(a[11]);
        at::Tensor out = at::empty({rows, gated ? n / 2 : n}, f32 ? x.options().dtype(at::kFloat) : x.options());
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(codes.data_ptr(), scales.data_ptr(), n, k, group, x.data_ptr(), rows, bias, f32 ? nullptr : out.data_ptr(),
                    f32 ? static_cast<float*>(out.data_ptr()) : nullptr, gated, act, -1, stream);
        }
        return rc != 0 ? PyLong_FromLong(rc) : wrap(out);
    });
}

typedef int (*LogprobsFn)(const void*, int, int, int, long long, const int*, int, float*, float*, int*, float*, int, int*, void*);

// logprobs(fn, logits, tokens, top, slices, status, stream, device): ops.token_logprobs, its four tensors as a tuple
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&](bool& called) -> PyObject* {
        const auto fn = reinterpret_cast<LogprobsFn>(address(a[0]));
        const int top = integer(a[3]), slices = integer(a[4]), device = integer(a[7]);
        const at::Tensor* x = on(tensor(a[1]), device);
        const at::Tensor& t = on(need(a[2], at::kInt, 1), device);
        if (!fn || !x || x->dim() != 2 || (x->size(1) > 1 && x->stride(1) != 1) || t.size(0) != x->size(0)) throw Bad{};
        const int64_t rows = size32(x->size(0)), vocab = size32(x->size(1));
        if (top < 0 || top > 64 || top > vocab) throw Bad{};
        const int type = type_code(*x);
        int* status = static_cast<int*>(address(a[5]));
        void* stream = address(a[6]);
        // (one allocation: the four are places of one storage)
        at::Tensor buf = at::empty({rows * (2 + 2LL * top)}, x->options().dtype(at::kFloat));
        float* p = static_cast<float*>(buf.data_ptr());
        auto place = [&](at::ScalarType of, int64_t offset, int64_t columns) {
            at::Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(of));
            part.unsafeGetTensorImpl()->set_storage_offset(offset);
            if (columns < 0) part.unsafeGetTensorImpl()->set_sizes_contiguous({rows});
            else part.unsafeGetTensorImpl()->set_sizes_contiguous({rows, columns});
            return part;
        };
        at::Tensor parts[4] = {place(at::kFloat, 0, -1), place(at::kFloat, rows, -1), place(at::kInt, 2 * rows, top), place(at::kFloat, (2 + top) * rows, top)};
        int rc;
        called = true;
        {
            Unlocked unlocked;
            rc = fn(x->data_ptr(), type, (int)rows, (int)vocab, x->stride(0), static_cast<const int*>(t.data_ptr()), top, p, p + rows,
                    reinterpret_cast<int*>(p + 2 * rows), p + (2 + top) * rows, slices, status, stream);
        }
        if (rc != 0) return PyLong_FromLong(rc);
        PyObject* all = PyTuple_New(4);
        for (int i = 0; all && i < 4; ++i) {
            PyObject* o = wrap(parts[i]);
            if (!o) { Py_DECREF(all); return nullptr; }
            PyTuple_SET_ITEM(all, i, o);
        }
        return all;
    });
}

PyMethodDef methods[] = {
    {"write8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write8)), METH_FASTCALL, "norm, rotation and the write to an 8-bit cache"},
    {"read8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read8)), METH_FASTCALL, "pages of an 8-bit cache as numbers"},
    {"attention8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention8)), METH_FASTCALL, "attention over an 8-bit cache"},
    {"int4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int4)), METH_FASTCALL, "a product of a few rows with a 4-bit weight"},
    {"logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logprobs)), METH_FASTCALL, "log probabilities of given tokens"},
    {"product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product)), METH_FASTCALL, "a fused product of a few rows"},
    {"shortconv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(shortconv)), METH_FASTCALL, "the gated short convolution"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "vapi_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_vapi_calls() { return PyModule_Create(&module); }
