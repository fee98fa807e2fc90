// Native half of unum_ops_b200/paged_cache.py: checks of arguments, allocation and the C ABI's calls.
//
// A decode step calls these operators for every layer, and its kernels run for a few microseconds; the same checks and
// allocations in Python, with the C ABI called through ctypes, took 24 us (append_cache) and 32 us (paged_attention) a
// call on the host, several times the kernels' own time.  Here a call takes its tensors as they are: no Python object is
// made on the way but the results.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <vector>

#include "../../include/unum_ops_b200.h"

namespace {

using at::Tensor;

// A refusal on its way to Python: the exception's type and message.
struct Refused {
    PyObject *type;
    std::string what;
};

struct Raised {};  // a Python exception that is set already

std::string text(const char *s) { return s; }
std::string text(int64_t x) { return std::to_string(x); }
std::string text(at::ScalarType x) { return c10::toString(x); }
std::string text(c10::Device x) { return x.str(); }
std::string text(at::IntArrayRef x) {
    std::string s = "[";
    for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + std::to_string(x[i]);
    return s + "]";
}

template <typename... A> [[noreturn]] void refuse(PyObject *type, const A &...a) {
    std::string s;
    (void)std::initializer_list<int>{(s += text(a), 0)...};
    throw Refused{type, s};
}

// Arguments in order, each taken by its name.
struct Args {
    PyObject *const *a;
    Tensor none;
    const Tensor &tensor(int i, const char *name) const {
        if (!THPVariable_Check(a[i])) refuse(PyExc_TypeError, name, " must be a tensor");
        return THPVariable_Unpack(a[i]);
    }
    const Tensor &optional_tensor(int i, const char *name) const { return a[i] == Py_None ? none : tensor(i, name); }
    int64_t integer(int i, const char *name) const {
        PyObject *v = PyNumber_Index(a[i]);
        const int64_t x = v ? PyLong_AsLongLong(v) : -1;
        Py_XDECREF(v);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            refuse(PyExc_TypeError, name, " must be an integer");
        }
        return x;
    }
    double number(int i, const char *name) const {
        const double x = PyFloat_AsDouble(a[i]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            refuse(PyExc_TypeError, name, " must be a number");
        }
        return x;
    }
    bool truth(int i) const {
        const int x = PyObject_IsTrue(a[i]);
        if (x < 0) throw Raised();
        return x == 1;
    }
};

// Tangents of forward mode count whatever the grad mode: torch.no_grad() does not turn them off.
void no_grad(std::initializer_list<const Tensor *> ts) {
    const bool backward = at::GradMode::is_enabled();
    for (const Tensor *t : ts) {
        if (!t->defined()) continue;
        if (backward && t->requires_grad())
            refuse(PyExc_NotImplementedError,
                   "the paged cache's operators have no backward pass: call them under torch.no_grad()");
        if (t->_fw_grad(/*level=*/0).defined())
            refuse(PyExc_NotImplementedError,
                   "the paged cache's operators have no forward-mode derivative: unpack dual tensors before the call");
    }
}

// Called after the other checks, so that those are the same on a machine without a GPU.
c10::Device on_one_gpu(std::initializer_list<const Tensor *> ts) {
    const Tensor &first = **ts.begin();
    for (const Tensor *t : ts) {
        if (!t->defined()) continue;
        if (!t->is_cuda())
            refuse(PyExc_ValueError, "unum_ops_b200 runs on CUDA tensors only; got a tensor on ", t->device());
        if (t->device() != first.device())
            refuse(PyExc_ValueError, "tensors on different devices: ", first.device(), " and ", t->device());
    }
    return first.device();
}

void check(int rc) {
    if (rc == UNUM_OK) return;
    if (rc == UNUM_ERR_INVALID) refuse(PyExc_ValueError, unum_last_error());
    if (rc == UNUM_ERR_UNSUPPORTED) refuse(PyExc_NotImplementedError, unum_last_error());
    refuse(PyExc_RuntimeError, "unum_ops_b200 error ", (int64_t)rc, ": ", unum_last_error());
}

// The stride of dim d in elements; 0 for a dim of one element (whose stride says nothing).
int64_t stride(const Tensor &t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Whether 16-byte loads can read the rows of a 3-d tensor of 2-byte elements.
bool has_rows16(const Tensor &t) {
    return t.stride(2) == 1 && (stride(t, 0) | stride(t, 1)) % 8 == 0 &&
           reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

Tensor rows16(const Tensor &t) { return has_rows16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether two elements may share memory (an expanded or an overlapping view).
bool overlaps(const Tensor &t) {
    if (t.is_contiguous()) return false;
    std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t reach = 0;
    for (const auto &d : dims) {
        if (d.first <= reach) return true;
        reach += (d.second - 1) * d.first;
    }
    return false;
}

// Whether the stretches of memory that two tensors span meet.
bool meet(const Tensor &a, const Tensor &b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    auto span = [](const Tensor &t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        return std::make_pair(at, at + (last + 1) * t.element_size());
    };
    const auto x = span(a), y = span(b);
    return x.first < y.second && y.first < x.second;
}

// Whether rows of two caches [n, Hk, D] meet; neither overlaps itself, and both have sizes and type alike.  Views that are
// interleaved in one buffer have one token stride, and then it is a question of the heads' distances modulo that stride.
// Interleaved with token strides of their own they count as meeting.
bool rows_meet(const Tensor &a, const Tensor &b) {
    if (!meet(a, b)) return false;
    const int64_t n = a.size(0), H = a.size(1), D = a.size(2), st = stride(a, 0), sa = stride(a, 1), sb = stride(b, 1);
    if (stride(b, 0) != st || (sa != sb && H > 256)) return true;
    const int64_t apart = (reinterpret_cast<intptr_t>(b.const_data_ptr()) - reinterpret_cast<intptr_t>(a.const_data_ptr())) /
                          (int64_t)a.element_size();
    auto hit = [&](int64_t d) {  // d + i * st, |i| < n, less than a row from 0
        int64_t i = st ? -d / st : 0;  // and its neighbours
        for (int64_t e = std::max(i - 1, 1 - n); e <= std::min(i + 1, n - 1); ++e)
            if (std::abs(d + e * st) < D) return true;
        return false;
    };
    for (int64_t h = 0; h < H; ++h)
        for (int64_t g = 0; g < (sa == sb && h ? 1 : H); ++g)  // with one head stride only the heads' difference counts
            if (hit(apart + g * sb - h * sa)) return true;
    return false;
}

// Ids and lengths in the kernels' type.  What 32 bits do not hold becomes their least or largest number, which is as far
// outside a table, a cache or a batch (a wrapped one could name another token); what is no number becomes -1.
Tensor to_i32(const Tensor &t) {
    const at::ScalarType type = t.scalar_type();
    if (type == at::kInt) return t;
    Tensor x = t;
    if (type == at::kUInt32 || type == at::kUInt64 || at::isFloatingType(type)) x = t.to(at::kDouble).nan_to_num(-1.0);
    if (x.scalar_type() == at::kDouble || type == at::kLong)
        x = x.clamp(std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max());
    return x.to(at::kInt);
}

Tensor as_i32(const Tensor &t) { return to_i32(t).contiguous(); }

void check_cache(const Tensor &k, const Tensor &v) {
    const char *name = "k_cache";
    for (const Tensor *c : {&k, &v}) {
        if (c->dim() != 3) refuse(PyExc_ValueError, name, " must be [n_tokens, Hk, D]; got ", c->sizes());
        if (c->scalar_type() != at::kBFloat16 && c->scalar_type() != at::kHalf)
            refuse(PyExc_ValueError, name, " must be bfloat16 or float16; got ", c->scalar_type());
        if (!has_rows16(*c))
            refuse(PyExc_ValueError, name, " must have contiguous, 16-byte aligned rows; got strides ", c->strides());
        name = "v_cache";
    }
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
        refuse(PyExc_ValueError, "k_cache and v_cache differ: ", k.sizes(), " ", k.scalar_type(), " and ", v.sizes(), " ",
               v.scalar_type());
}

void check_table(const Tensor &t, int64_t page_size) {
    if (t.dim() != 2) refuse(PyExc_ValueError, "block_table must be [B, n_pages]; got ", t.sizes());
    if (page_size < 1 || (page_size & (page_size - 1)) || page_size > 65536)
        refuse(PyExc_ValueError, "page_size must be a power of two up to 65536; got ", page_size);
}

Tensor table_i32(const Tensor &t) {
    const Tensor x = to_i32(t);
    return x.stride(1) == 1 || x.size(1) < 2 ? x : x.contiguous();
}

void written(const Tensor &t) {  // for whoever has saved it
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Runs f while other Python threads run: an allocation or a launch may wait for the device.  f makes no Python object.
template <typename F> auto released(const F &f) {
    struct Free {
        PyThreadState *state = PyEval_SaveThread();
        ~Free() { PyEval_RestoreThread(state); }
    } free;
    return f();
}

void *stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

void append(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &table, const Tensor &bs,
            const Tensor &pos, int64_t page) {
    no_grad({&k, &v, &kc, &vc});
    check_cache(kc, vc);
    if (k.dim() != 3 || k.sizes() != v.sizes() || k.size(1) != kc.size(1) || k.size(2) != kc.size(2))
        refuse(PyExc_ValueError, "k and v must be [T, ", kc.size(1), ", ", kc.size(2), "] like the cache's rows; got ",
               k.sizes(), " and ", v.sizes());
    if (k.scalar_type() != kc.scalar_type() || v.scalar_type() != kc.scalar_type())
        refuse(PyExc_ValueError, "k and v must have the cache's dtype ", kc.scalar_type(), "; got ", k.scalar_type(), " and ",
               v.scalar_type());
    if (overlaps(kc) || overlaps(vc) || rows_meet(kc, vc))
        refuse(PyExc_ValueError, "k_cache and v_cache are written to: their rows must not share memory");
    if (meet(k, kc) || meet(k, vc) || meet(v, kc) || meet(v, vc))
        refuse(PyExc_ValueError, "k and v must not lie in the memory of k_cache and v_cache");
    const int64_t T = k.size(0);
    if (bs.numel() != T || pos.numel() != T)
        refuse(PyExc_ValueError, "token_to_bs and token_pos_in_bs must have one entry for each of ", T, " tokens; got ",
               bs.numel(), " and ", pos.numel());
    check_table(table, page);
    const c10::Device dev = on_one_gpu({&k, &v, &kc, &vc, &table, &bs, &pos});
    if (k.numel() == 0) return;
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor k_ = rows16(k), v_ = rows16(v), t = table_i32(table), bs_ = as_i32(bs), pos_ = as_i32(pos);
    check(unum_cache_append(k_.const_data_ptr(), v_.const_data_ptr(), T, k_.size(1), k_.size(2), stride(k_, 0), stride(k_, 1),
                            stride(v_, 0), stride(v_, 1), kc.data_ptr(), vc.data_ptr(), kc.size(0), stride(kc, 0),
                            stride(kc, 1), stride(vc, 0), stride(vc, 1), t.const_data_ptr<int32_t>(), t.size(0), t.size(1),
                            t.stride(0), page, bs_.const_data_ptr<int32_t>(), pos_.const_data_ptr<int32_t>(),
                            stream_of(dev)));
    written(kc);
    written(vc);
}

// append_cache(k, v, k_cache, v_cache, block_table, token_to_bs, token_pos_in_bs, page_size)
PyObject *append_cache(const Args &a) {
    const Tensor &k = a.tensor(0, "k"), &v = a.tensor(1, "v"), &kc = a.tensor(2, "k_cache"), &vc = a.tensor(3, "v_cache");
    const Tensor &table = a.tensor(4, "block_table"), &bs = a.tensor(5, "token_to_bs"), &pos = a.tensor(6, "token_pos_in_bs");
    const int64_t page = a.integer(7, "page_size");
    released([&] { append(k, v, kc, vc, table, bs, pos, page); });
    Py_RETURN_NONE;
}

// The output and, where it is asked for, the lse.
std::pair<Tensor, Tensor> attend(const Tensor &q, const Tensor &kc, const Tensor &vc, const Tensor &table, const Tensor &lens,
                                 int64_t page, std::optional<int64_t> max_seqlen, std::optional<double> softmax_scale,
                                 const Tensor &weights, bool return_lse) {
    no_grad({&q, &kc, &vc, &weights});
    check_cache(kc, vc);
    if (q.dim() != 3 || q.size(2) != kc.size(2))
        refuse(PyExc_ValueError, "q must be [B, Hq, ", kc.size(2), "]; got ", q.sizes());
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), Hk = kc.size(1);
    if (q.scalar_type() != kc.scalar_type())
        refuse(PyExc_ValueError, "q must have the cache's dtype ", kc.scalar_type(), "; got ", q.scalar_type());
    if (Hk == 0 || Hq == 0 || Hq % Hk)
        refuse(PyExc_ValueError, Hq, " query heads are no multiple of ", Hk, " kv heads");
    check_table(table, page);
    if (table.size(0) != B || lens.numel() != B)
        refuse(PyExc_ValueError, "block_table and seqlens must have one row for each of ", B, " sequences; got ",
               table.size(0), " and ", lens.numel());
    int64_t max_len = table.size(1) * page;
    if (max_seqlen) max_len = std::min(max_len, *max_seqlen);
    if (max_len < 0) refuse(PyExc_ValueError, "max_seqlen must not be negative; got ", max_len);
    if (weights.defined()) {
        if (weights.dim() != 3 || weights.size(0) != B || weights.size(1) != Hk || weights.size(2) < max_len)
            refuse(PyExc_ValueError, "weights must be [", B, ", ", Hk, ", >= ", max_len, "]; got ", weights.sizes());
        if (weights.scalar_type() != at::kFloat || (weights.stride(2) != 1 && weights.size(2) > 1) || overlaps(weights))
            refuse(PyExc_ValueError, "weights must be float32 with contiguous rows that share no memory");
    }
    const double scale = softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)D);
    const c10::Device dev = on_one_gpu({&q, &kc, &vc, &table, &lens, &weights});
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    Tensor lse;
    if (return_lse) lse = at::empty({B, Hq}, q.options().dtype(at::kFloat));
    if (B) {
        const Tensor q_ = rows16(q), t = table_i32(table), lens_ = as_i32(lens);
        const size_t bytes = unum_paged_attention_workspace_size(B, Hq, Hk, D, max_len, weights.defined());
        // a call's own: calls on other streams, or of other graphs, may run at the same time
        const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
        check(unum_paged_attention(
            q_.const_data_ptr(), B, Hq, D, stride(q_, 0), stride(q_, 1), kc.const_data_ptr(), vc.const_data_ptr(),
            q.scalar_type() == at::kHalf ? UNUM_DTYPE_F16 : UNUM_DTYPE_BF16, kc.size(0), Hk, stride(kc, 0), stride(kc, 1),
            stride(vc, 0), stride(vc, 1), t.const_data_ptr<int32_t>(), t.size(1), t.stride(0), page,
            lens_.const_data_ptr<int32_t>(), max_len, (float)scale, out.data_ptr(), lse.defined() ? lse.data_ptr<float>() : nullptr,
            weights.defined() ? weights.data_ptr<float>() : nullptr, weights.defined() ? weights.stride(0) : 0,
            weights.defined() ? weights.stride(1) : 0, ws.get(), bytes, stream_of(dev)));
        if (weights.defined()) written(weights);
    }
    return {out, lse};
}

// paged_attention(q, k_cache, v_cache, block_table, seqlens, page_size, max_seqlen, softmax_scale, weights, return_lse)
PyObject *paged_attention(const Args &a) {
    const Tensor &q = a.tensor(0, "q"), &kc = a.tensor(1, "k_cache"), &vc = a.tensor(2, "v_cache");
    const Tensor &table = a.tensor(3, "block_table"), &lens = a.tensor(4, "seqlens");
    const int64_t page = a.integer(5, "page_size");
    std::optional<int64_t> max_seqlen;
    if (a.a[6] != Py_None) max_seqlen = a.integer(6, "max_seqlen");
    std::optional<double> scale;
    if (a.a[7] != Py_None) scale = a.number(7, "softmax_scale");
    const Tensor &weights = a.optional_tensor(8, "weights");
    const bool return_lse = a.truth(9);
    const auto [out, lse] =
        released([&] { return attend(q, kc, vc, table, lens, page, max_seqlen, scale, weights, return_lse); });
    if (!lse.defined()) return THPVariable_Wrap(out);
    return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
}

std::array<Tensor, 4> evict(const Tensor &table, const Tensor &lens, const Tensor &weights, int64_t budget, int64_t init,
                            int64_t local, int64_t page) {
    no_grad({&weights});
    check_table(table, page);
    const int64_t B = table.size(0), n_pages = table.size(1);
    if (lens.numel() != B)
        refuse(PyExc_ValueError, "seqlens must have one entry for each of ", B, " sequences; got ", lens.numel());
    if (weights.dim() != 3 || weights.size(0) != B || weights.size(1) < 1 || weights.size(2) != n_pages * page)
        refuse(PyExc_ValueError, "weights must be [", B, ", Hk, ", n_pages * page, "]; got ", weights.sizes());
    if (weights.scalar_type() != at::kFloat)
        refuse(PyExc_ValueError, "weights must be float32; got ", weights.scalar_type());
    if (local < 1 || init < 0 || budget < 0 || budget - init < local)
        refuse(PyExc_ValueError, "need init_pages >= 0, local_pages >= 1 and budget >= their sum; got budget ", budget,
               ", init_pages ", init, ", local_pages ", local);
    const c10::Device dev = on_one_gpu({&table, &lens, &weights});
    const c10::cuda::CUDAGuard guard(dev);
    const auto ints = weights.options().dtype(at::kInt);
    const Tensor new_table = at::empty({B, n_pages}, ints), new_lens = at::empty({B}, ints);
    const Tensor new_w = at::empty(weights.sizes(), weights.options().memory_format(at::MemoryFormat::Contiguous));
    const Tensor gone = at::empty({B, n_pages}, ints);
    if (B) {
        const Tensor t = table_i32(table), lens_ = as_i32(lens);
        const Tensor w = weights.stride(2) == 1 || weights.size(2) < 2 ? weights : weights.contiguous();
        check(unum_cache_evict(t.const_data_ptr<int32_t>(), B, n_pages, t.stride(0), lens_.const_data_ptr<int32_t>(),
                               w.const_data_ptr<float>(), w.size(1), w.stride(0), w.stride(1), page, budget, init, local,
                               new_table.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), new_w.data_ptr<float>(),
                               gone.data_ptr<int32_t>(), stream_of(dev)));
    }
    return {new_table, new_lens, new_w, gone};
}

// evict_cache(block_table, seqlens, weights, budget, init_pages, local_pages, page_size)
PyObject *evict_cache(const Args &a) {
    const Tensor &table = a.tensor(0, "block_table"), &lens = a.tensor(1, "seqlens"), &weights = a.tensor(2, "weights");
    const int64_t budget = a.integer(3, "budget"), init = a.integer(4, "init_pages"), local = a.integer(5, "local_pages");
    const int64_t page = a.integer(6, "page_size");
    const auto r = released([&] { return evict(table, lens, weights, budget, init, local, page); });
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(r[0]), THPVariable_Wrap(r[1]), THPVariable_Wrap(r[2]),
                         THPVariable_Wrap(r[3]));
}

template <PyObject *(*kFn)(const Args &), int kArgs>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    try {
        if (n != kArgs) refuse(PyExc_TypeError, "expected ", (int64_t)kArgs, " arguments, got ", (int64_t)n);
        return kFn(Args{args, {}});
    } catch (const Raised &) {
    } catch (const Refused &r) {
        PyErr_SetString(r.type, r.what.c_str());
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *torch = PyImport_ImportModule("torch");
        PyObject *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (type) PyErr_SetString(type, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(entry<name, n>), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(append_cache, 8), ENTRY(paged_attention, 10), ENTRY(evict_cache, 7),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
