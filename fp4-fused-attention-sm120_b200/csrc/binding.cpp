// binding.cpp -- the serving calls' way from torch tensors to the C ABI
// (fp4attn_b200._native; rotary.py and paged.py are its only callers).
//
// A decode step makes these calls once a layer and token.  Checking five
// tensors, allocating two and passing 25 arguments through ctypes took 15 us of
// host time a call, several times what the kernels take; here it is two to
// four.  The functions are those of the shared library, by the addresses that
// the Python side looked up; there is no arithmetic here.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <optional>
#include <string>
#include <vector>

#include "../../include/fp4attn.h"

namespace {

struct Calls {
    decltype(&fp4attn_rotary) rotary;
    decltype(&fp4attn_cache_append) cache_append;
    decltype(&fp4attn_cache_gather) cache_gather;
    decltype(&fp4attn_paged_attention_workspace_size) workspace_size;
    decltype(&fp4attn_paged_attention) paged_attention;
    decltype(&fp4attn_copy_pages) copy_pages;
} g;
PyObject* g_check = nullptr;  // check(status, name): raises for a status that is not OK

using at::Tensor;

#define REFUSE(cond, ...)                                \
    do {                                                 \
        if (cond) {                                      \
            PyErr_Format(PyExc_ValueError, __VA_ARGS__); \
            return nullptr;                              \
        }                                                \
    } while (0)

// A tensor argument: null (with the error set) if it is none.
const Tensor* tensor(PyObject* o, const char* name)
{
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
        return nullptr;
    }
    return &THPVariable_Unpack(o);
}

#define TENSOR(var, object, name)             \
    const Tensor* var = tensor(object, name); \
    if (!var) return nullptr

int code_of(at::ScalarType t) { return t == at::kHalf ? FP4ATTN_F16 : t == at::kFloat ? FP4ATTN_F32 : -1; }

#define DTYPE(var, type)                                                                            \
    const int var = code_of(type);                                                                  \
    if (var < 0) {                                                                                  \
        PyErr_Format(PyExc_TypeError, "unsupported dtype %s; use float16 or float32", toString(type)); \
        return nullptr;                                                                             \
    }

// A float16 / float32 dtype argument, or `otherwise` for None.
bool dtype_arg(PyObject* o, at::ScalarType otherwise, at::ScalarType* out)
{
    if (o == Py_None) {
        *out = otherwise;
    } else if (THPDtype_Check(o)) {
        *out = reinterpret_cast<THPDtype*>(o)->scalar_type;
    } else {
        PyErr_SetString(PyExc_TypeError, "dtype must be a torch.dtype");
        return false;
    }
    return true;
}

bool good_index(const Tensor& t, const at::Device& d, const char* name)
{
    if (t.scalar_type() == at::kInt && t.device() == d) return true;
    PyErr_Format(PyExc_ValueError, "%s must be an int32 tensor on %s", name, d.str().c_str());
    return false;
}

bool good_vector(const Tensor& t, int64_t n, const at::Device& d, const char* name)
{
    if (!good_index(t, d, name)) return false;
    if (t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1)) return true;
    PyErr_Format(PyExc_ValueError, "%s must be a contiguous int32 [%lld] tensor", name, static_cast<long long>(n));
    return false;
}

// [tokens, heads, head_dim] rows (heads < 0: any number).
bool good_rows(const Tensor& t, int64_t tokens, int heads, int dim, at::ScalarType type, const at::Device& d, const char* name)
{
    if (t.dim() == 3 && t.size(0) == tokens && (heads < 0 || t.size(1) == heads) && t.size(2) == dim && t.device() == d &&
        t.scalar_type() == type && t.stride(2) == 1)
        return true;
    PyErr_Format(PyExc_ValueError, "%s must be a [%lld, %s, %d] %s tensor on %s with a contiguous last dimension", name,
                 static_cast<long long>(tokens), heads < 0 ? "heads" : std::to_string(heads).c_str(), dim, toString(type),
                 d.str().c_str());
    return false;
}

struct Table {
    const int32_t* pages;
    int64_t stride;
    int seqs, max_pages;
};
bool good_table(const Tensor& t, const at::Device& d, Table* out)
{
    if (!good_index(t, d, "block_table")) return false;
    if (t.dim() != 2 || t.size(1) < 1 || t.stride(1) != 1 || t.size(0) > INT_MAX || t.size(1) > INT_MAX) {
        PyErr_SetString(PyExc_ValueError, "block_table must be [sequences, pages] with contiguous rows");
        return false;
    }
    *out = Table{t.const_data_ptr<int32_t>(), t.size(0) > 1 ? t.stride(0) : t.size(1), static_cast<int>(t.size(0)),
                 static_cast<int>(t.size(1))};
    return true;
}

struct Angles {
    const float* table = nullptr;
    int rotary_dim = 0;
    int64_t positions = 0;
};
bool good_angles(PyObject* o, const at::Device& d, int64_t head_dim, Angles* out)
{
    if (o == Py_None) return true;
    const Tensor* t = tensor(o, "table");
    if (!t) return false;
    if (t->dim() != 3 || t->size(2) != 2 || t->scalar_type() != at::kFloat || t->device() != d || !t->is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "table must be a contiguous float32 [positions, rotary_dim / 2, 2] tensor on %s", d.str().c_str());
        return false;
    }
    if (2 * t->size(1) > head_dim) {
        PyErr_Format(PyExc_ValueError, "the table's rotary_dim %lld exceeds head_dim %lld", static_cast<long long>(2 * t->size(1)),
                     static_cast<long long>(head_dim));
        return false;
    }
    if (t->numel() == 0) {  // (a null pointer would read as no table at all)
        PyErr_SetString(PyExc_ValueError, "the table is empty");
        return false;
    }
    *out = Angles{t->const_data_ptr<float>(), static_cast<int>(2 * t->size(1)), t->size(0)};
    return true;
}

Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Device& d)
{
    return at::detail::empty_cuda(sizes, type, d, std::nullopt);
}

void* stream_of(const at::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// Whether the call went well; else the Python side's check raises.
bool went(int status, const char* name)
{
    if (status == FP4ATTN_OK) return true;
    PyObject* r = PyObject_CallFunction(g_check, "is", status, name);
    if (r) {  // (it always raises)
        Py_DECREF(r);
        PyErr_Format(PyExc_RuntimeError, "%s: status %d", name, status);
    }
    return false;
}

#define ARGS(n, name)                                                          \
    if (argc != n) {                                                           \
        PyErr_Format(PyExc_TypeError, name " takes %d arguments, got %zd", n, argc); \
        return nullptr;                                                        \
    }

// The cache's description and device: (address of an fp4attn_cache, device index).
#define CACHE(object, index)                                                                  \
    const auto* cache = static_cast<const fp4attn_cache*>(PyLong_AsVoidPtr(object));          \
    const at::Device device(at::kCUDA, static_cast<at::DeviceIndex>(PyLong_AsLong(index)));   \
    if (PyErr_Occurred()) return nullptr

// One multiple of a stride, least to most, out of a sum of them.
struct Term {
    int64_t stride, least, most;
};

// Whether start + sum_k m_k stride_k can lie between lo and hi (both excluded)
// for m_k in [least, most], not all of them zero if `moved`.  Strides in falling
// order, positive; with those of an ordinary view few multiples of each come into
// question.  A search that takes too long counts as yes.
bool meets(const std::vector<Term>& t, size_t k, int64_t start, int64_t lo, int64_t hi, bool moved, int& steps)
{
    if (++steps > 20000) return true;
    if (k == t.size()) return !moved && lo < start && start < hi;
    int64_t below = 0, above = 0;  // what the terms behind this one reach
    for (size_t i = k + 1; i < t.size(); i++) {
        below += t[i].least * t[i].stride;
        above += t[i].most * t[i].stride;
    }
    const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t first = std::max(t[k].least, floor_div(lo - above - start, t[k].stride) + 1);
    const int64_t last = std::min(t[k].most, -floor_div(start + below - hi, t[k].stride) - 1);
    for (int64_t m = first; m <= last; m++)
        if (meets(t, k + 1, start + m * t[k].stride, lo, hi, moved && m == 0, steps)) return true;
    return false;
}

bool meets(std::vector<Term>& t, int64_t start, int64_t lo, int64_t hi, bool moved)
{
    std::sort(t.begin(), t.end(), [](const Term& a, const Term& b) { return a.stride > b.stride; });
    int steps = 0;
    return meets(t, 0, start, lo, hi, moved, steps);
}

// Checks `out`, which a call reads `in` to write, of one shape and both with
// contiguous rows: it may be `in` or lie between its rows, but neither have
// elements in common with it otherwise nor with itself.  (Both are mostly slices
// of a wider projection, so this is decided from the strides.)  Its version is
// moved on, so that autograd notices where it had kept the old contents.
void writes_over(const Tensor& out, const Tensor& in, const char* name)
{
    const int64_t rows = out.dim() - 1, oe = out.element_size(), ie = in.element_size();
    if (out.numel() > 0) {
        std::vector<Term> self, both;
        bool in_place = out.const_data_ptr() == in.const_data_ptr() && oe == ie;
        for (int64_t k = 0; k < rows; k++) {
            const int64_t n = out.size(k), os = out.stride(k) * oe, is = in.stride(k) * ie;
            if (n == 1) continue;
            TORCH_CHECK_VALUE(os > 0, "elements of out share memory");
            self.push_back({os, 1 - n, n - 1});
            in_place = in_place && os == is;
            if (os == is) {
                both.push_back({os, 1 - n, n - 1});
            } else {
                both.push_back({os, 0, n - 1});
                if (is > 0) both.push_back({is, 1 - n, 0});
            }
        }
        const int64_t out_row = out.size(rows) * oe, in_row = in.size(rows) * ie;
        TORCH_CHECK_VALUE(!meets(self, 0, -out_row, out_row, true), "elements of out share memory");
        const int64_t apart = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out.const_data_ptr()) -
                                                   reinterpret_cast<uintptr_t>(in.const_data_ptr()));
        TORCH_CHECK_VALUE(in_place || !meets(both, apart, -out_row, in_row, false), "out lies partly over ", name);
    }
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// x turned into `out` (undefined: a new tensor); throws on a bad argument.
Tensor rotary(const Tensor& x, const Tensor& table, const std::optional<Tensor>& positions, bool interleaved, bool inverse,
              Tensor out)
{
    TORCH_CHECK_VALUE(x.dim() == 4 && x.is_cuda() && x.stride(3) == 1,
                      "x must be a [batch, heads, seq, head_dim] CUDA tensor with a contiguous last dimension");
    const at::Device device = x.device();
    const at::ScalarType type = x.scalar_type();
    const int code = code_of(type);
    TORCH_CHECK_TYPE(code >= 0, "unsupported dtype ", toString(type), "; use float16 or float32");
    const int64_t B = x.size(0), H = x.size(1), S = x.size(2), D = x.size(3);
    TORCH_CHECK_VALUE(B <= INT_MAX && H <= INT_MAX && S <= INT_MAX && D <= INT_MAX, "x is too large");
    TORCH_CHECK_VALUE(table.dim() == 3 && table.size(2) == 2 && table.scalar_type() == at::kFloat && table.device() == device &&
                          table.is_contiguous(),
                      "table must be a contiguous float32 [positions, rotary_dim / 2, 2] tensor on ", device.str());
    TORCH_CHECK_VALUE(2 * table.size(1) <= D, "the table's rotary_dim ", 2 * table.size(1), " exceeds head_dim ", D);
    const int32_t* at = nullptr;
    int64_t at_stride = 0;
    if (positions) {
        const Tensor& p = *positions;
        TORCH_CHECK_VALUE(p.scalar_type() == at::kInt && p.device() == device, "positions must be an int32 tensor on ", device.str());
        const bool each = p.dim() == 2 && p.size(0) == B && p.size(1) == S;
        TORCH_CHECK_VALUE(each || (p.dim() == 1 && p.size(0) == S), "positions must be [seq] or [batch, seq]");
        TORCH_CHECK_VALUE(S < 2 || p.stride(-1) == 1, "positions must be contiguous along seq");
        at = p.const_data_ptr<int32_t>();
        at_stride = each ? p.stride(0) : 0;
    }
    const c10::cuda::CUDAGuard guard(device);
    const bool given = out.defined();
    if (!given) out = make(x.sizes(), type, device);
    else
        TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == type && out.device() == device && out.stride(3) == 1,
                          "out must have x's shape, dtype and device, and a contiguous last dimension");
    if (given) writes_over(out, x, "x");
    const int64_t xs[3] = {x.stride(0), x.stride(1), x.stride(2)}, os[3] = {out.stride(0), out.stride(1), out.stride(2)};
    const int status = g.rotary(x.const_data_ptr(), out.mutable_data_ptr(), code, B, H, S, D, xs, os, table.const_data_ptr<float>(),
                                2 * table.size(1), table.size(0), at, at_stride, interleaved, inverse, stream_of(device));
    if (status != FP4ATTN_OK) {
        pybind11::gil_scoped_acquire gil;  // (a backward pass runs without it)
        went(status, "fp4attn_rotary");
        throw python_error();
    }
    return out;
}

// A tensor or None.
bool optional_tensor(PyObject* o, const char* name, std::optional<Tensor>* out)
{
    if (o == Py_None) return true;
    const Tensor* t = tensor(o, name);
    if (t) *out = *t;
    return t != nullptr;
}

PyObject* native_rotary(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(6, "rotary");  // x, table, positions, interleaved, inverse, out
    TENSOR(x, args[0], "x");
    TENSOR(table, args[1], "table");
    std::optional<Tensor> positions, out;
    if (!optional_tensor(args[2], "positions", &positions) || !optional_tensor(args[5], "out", &out)) return nullptr;
    const Tensor y = rotary(*x, *table, positions, PyObject_IsTrue(args[3]), PyObject_IsTrue(args[4]), out.value_or(Tensor()));
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// The rotation under autograd: the gradient turns back by the same angles, by
// this same function, so that it can be differentiated in turn.
struct Rotary : torch::autograd::Function<Rotary> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& table,
                          const std::optional<Tensor>& positions, bool interleaved, bool inverse)
    {
        ctx->save_for_backward({table, positions.value_or(Tensor())});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        return rotary(x, table, positions, interleaved, inverse, Tensor());
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        Tensor dy = grads[0];
        if (dy.stride(3) != 1) dy = dy.contiguous();
        const std::optional<Tensor> positions = saved[1].defined() ? std::optional<Tensor>(saved[1]) : std::nullopt;
        return {apply(dy, saved[0], positions, ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool()),
                Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

PyObject* native_rotary_embedding(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(4, "rotary_embedding");  // x, table, positions, interleaved
    TENSOR(x, args[0], "x");
    TENSOR(table, args[1], "table");
    std::optional<Tensor> positions;
    if (!optional_tensor(args[2], "positions", &positions)) return nullptr;
    REFUSE(table->requires_grad(), "the table has no gradient");
    return THPVariable_Wrap(Rotary::apply(*x, *table, positions, static_cast<bool>(PyObject_IsTrue(args[3])), false));
    END_HANDLE_TH_ERRORS
}

PyObject* native_cache_append(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(11, "cache_append");  // cache, device, K, V, block_table, positions, seq_ids, Q, table, interleaved, scale rule
    CACHE(args[0], args[1]);
    TENSOR(K, args[2], "K");
    TENSOR(V, args[3], "V");
    TENSOR(block_table, args[4], "block_table");
    TENSOR(positions, args[5], "positions");
    const at::ScalarType type = K->scalar_type();
    DTYPE(code, type);
    const int64_t tokens = K->dim() ? K->size(0) : 0;
    REFUSE(tokens > INT_MAX, "too many tokens");
    const int dim = cache->head_dim;
    if (!good_rows(*K, tokens, cache->kv_heads, dim, type, device, "K") ||
        !good_rows(*V, tokens, cache->kv_heads, dim, type, device, "V"))
        return nullptr;
    Table t;
    Angles angles;
    if (!good_table(*block_table, device, &t) || !good_vector(*positions, tokens, device, "positions") ||
        !good_angles(args[8], device, dim, &angles))
        return nullptr;
    const int32_t* seq_ids = nullptr;
    if (args[6] != Py_None) {
        TENSOR(ids, args[6], "seq_ids");
        if (!good_vector(*ids, tokens, device, "seq_ids")) return nullptr;
        seq_ids = ids->const_data_ptr<int32_t>();
    }
    const c10::cuda::CUDAGuard guard(device);
    Tensor out;
    const void* q = nullptr;
    int64_t qs[2] = {0, 0};
    int q_heads = 0;
    if (args[7] != Py_None) {
        TENSOR(Q, args[7], "Q");
        if (!good_rows(*Q, tokens, -1, dim, type, device, "Q")) return nullptr;
        out = make(Q->sizes(), type, device);
        q = Q->const_data_ptr();
        qs[0] = Q->stride(0);
        qs[1] = Q->stride(1);
        REFUSE(Q->size(1) > INT_MAX, "Q is too large");
        q_heads = static_cast<int>(Q->size(1));
    }
    const long rule = PyLong_AsLong(args[10]);
    const int64_t ks[2] = {K->stride(0), K->stride(1)}, vs[2] = {V->stride(0), V->stride(1)};
    if (!went(g.cache_append(cache, K->const_data_ptr(), V->const_data_ptr(), q, q ? out.mutable_data_ptr() : nullptr, code,
                             tokens, q_heads, ks, vs, qs, t.pages, t.stride, t.seqs, t.max_pages, seq_ids,
                             positions->const_data_ptr<int32_t>(), angles.table, angles.rotary_dim, angles.positions,
                             PyObject_IsTrue(args[9]), rule, stream_of(device)),
              "fp4attn_cache_append"))
        return nullptr;
    if (args[7] == Py_None) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyObject* native_cache_gather(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(8, "cache_gather");  // cache, device, block_table, starts, lengths, max_length, heads, dtype
    CACHE(args[0], args[1]);
    TENSOR(block_table, args[2], "block_table");
    TENSOR(lengths, args[4], "lengths");
    Table t;
    if (!good_table(*block_table, device, &t) || !good_vector(*lengths, t.seqs, device, "lengths")) return nullptr;
    const int32_t* starts = nullptr;
    if (args[3] != Py_None) {
        TENSOR(s, args[3], "starts");
        if (!good_vector(*s, t.seqs, device, "starts")) return nullptr;
        starts = s->const_data_ptr<int32_t>();
    }
    const long most = PyLong_AsLong(args[5]);
    const long heads = args[6] == Py_None ? cache->kv_heads : PyLong_AsLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    REFUSE(most < 0 || most > INT_MAX || heads < 1 || heads > INT_MAX, "max_length must be >= 0 and heads >= 1");
    at::ScalarType type;
    if (!dtype_arg(args[7], at::kHalf, &type)) return nullptr;
    DTYPE(code, type);
    const c10::cuda::CUDAGuard guard(device);
    const int64_t shape[4] = {t.seqs, heads, most, cache->head_dim};
    Tensor K = make(shape, type, device), V = make(shape, type, device);
    if (!went(g.cache_gather(cache, t.pages, t.stride, t.seqs, t.max_pages, starts, lengths->const_data_ptr<int32_t>(), most, heads,
                             K.mutable_data_ptr(), V.mutable_data_ptr(), code, stream_of(device)),
              "fp4attn_cache_gather"))
        return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(K), THPVariable_Wrap(V));
    END_HANDLE_TH_ERRORS
}

PyObject* native_attend(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(11, "attend");  // Q, cache, device, block_table, seq_lens, scale, scale rule, out_dtype, out, with lse, workspace
    TENSOR(Q, args[0], "Q");
    CACHE(args[1], args[2]);
    TENSOR(block_table, args[3], "block_table");
    TENSOR(seq_lens, args[4], "seq_lens");
    const at::ScalarType type = Q->scalar_type();
    DTYPE(code, type);
    const int64_t B = Q->dim() ? Q->size(0) : 0;
    if (!good_rows(*Q, B, -1, cache->head_dim, type, device, "Q")) return nullptr;
    const int64_t H = Q->size(1);
    REFUSE(B > INT_MAX || H > INT_MAX, "Q is too large");
    Table t;
    if (!good_table(*block_table, device, &t)) return nullptr;
    REFUSE(t.seqs != B, "block_table has %d rows for %lld queries", t.seqs, static_cast<long long>(B));
    if (!good_vector(*seq_lens, B, device, "seq_lens")) return nullptr;
    const double scale = args[5] == Py_None ? 0.0 : PyFloat_AsDouble(args[5]);
    const long rule = PyLong_AsLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType out_type;
    if (!dtype_arg(args[7], type, &out_type)) return nullptr;
    const c10::cuda::CUDAGuard guard(device);
    Tensor out, lse, workspace;
    if (args[8] == Py_None) {
        DTYPE(checked, out_type);
        (void)checked;
        out = make(Q->sizes(), out_type, device);
    } else {
        TENSOR(o, args[8], "out");
        REFUSE(o->sizes() != Q->sizes() || !o->is_contiguous() || o->device() != device ||
                   (args[7] != Py_None && o->scalar_type() != out_type),
               "out must be contiguous with Q's shape, on its device");
        out = *o;
        writes_over(out, *Q, "Q");
    }
    DTYPE(out_code, out.scalar_type());
    const bool with_lse = PyObject_IsTrue(args[9]);
    if (with_lse) lse = make({B, H}, at::kFloat, device);
    if (args[10] == Py_None) {
        const size_t size = g.workspace_size(B, H, cache->kv_heads, cache->head_dim);
        workspace = make({static_cast<int64_t>(size ? size : 1)}, at::kByte, device);
    } else {
        TENSOR(w, args[10], "workspace");
        REFUSE(w->device() != device || w->scalar_type() != at::kByte || !w->is_contiguous(),
               "workspace must be a contiguous uint8 tensor on Q's device");
        workspace = *w;
    }
    const int64_t qs[2] = {Q->stride(0), Q->stride(1)};
    if (!went(g.paged_attention(cache, Q->const_data_ptr(), out.mutable_data_ptr(),
                                with_lse ? lse.mutable_data_ptr<float>() : nullptr, code, out_code, B, H, qs, t.pages, t.stride,
                                t.max_pages, seq_lens->const_data_ptr<int32_t>(), static_cast<float>(scale), rule,
                                workspace.mutable_data_ptr(), workspace.numel(), stream_of(device)),
              "fp4attn_paged_attention"))
        return nullptr;
    PyObject* o;
    if (args[8] != Py_None) {
        o = args[8];
        Py_INCREF(o);
    } else {
        o = THPVariable_Wrap(out);
    }
    if (!with_lse) return o;
    return Py_BuildValue("(NN)", o, THPVariable_Wrap(lse));
    END_HANDLE_TH_ERRORS
}

PyObject* native_copy_pages(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    HANDLE_TH_ERRORS
    ARGS(4, "copy_pages");  // list of cache addresses, device, src, dst
    TENSOR(src, args[2], "src");
    TENSOR(dst, args[3], "dst");
    const at::Device device(at::kCUDA, static_cast<at::DeviceIndex>(PyLong_AsLong(args[1])));
    if (PyErr_Occurred()) return nullptr;
    for (const Tensor* t : {src, dst})
        REFUSE(t->is_cuda() || t->scalar_type() != at::kInt || t->dim() != 1 || !t->is_contiguous(),
               "src and dst must be page numbers in host memory");
    REFUSE(src->numel() != dst->numel(), "src and dst differ in length");
    REFUSE(src->numel() > INT_MAX, "too many pages");
    std::vector<fp4attn_cache> caches;
    const Py_ssize_t n = PyList_Size(args[0]);
    for (Py_ssize_t i = 0; i < n; i++) {
        const auto* c = static_cast<const fp4attn_cache*>(PyLong_AsVoidPtr(PyList_GET_ITEM(args[0], i)));
        if (PyErr_Occurred()) return nullptr;
        caches.push_back(*c);
    }
    if (PyErr_Occurred()) return nullptr;
    const c10::cuda::CUDAGuard guard(device);
    if (!went(g.copy_pages(caches.data(), static_cast<int>(caches.size()), src->const_data_ptr<int32_t>(),
                           dst->const_data_ptr<int32_t>(), static_cast<int>(src->numel()), stream_of(device)),
              "fp4attn_copy_pages"))
        return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// bind(check, addresses of the six functions in the order of Calls)
PyObject* native_bind(PyObject*, PyObject* const* args, Py_ssize_t argc)
{
    ARGS(7, "bind");
    void* p[6];
    for (int i = 0; i < 6; i++) p[i] = PyLong_AsVoidPtr(args[1 + i]);
    if (PyErr_Occurred()) return nullptr;
    Py_XDECREF(g_check);
    Py_INCREF(args[0]);
    g_check = args[0];
    g.rotary = reinterpret_cast<decltype(g.rotary)>(p[0]);
    g.cache_append = reinterpret_cast<decltype(g.cache_append)>(p[1]);
    g.cache_gather = reinterpret_cast<decltype(g.cache_gather)>(p[2]);
    g.workspace_size = reinterpret_cast<decltype(g.workspace_size)>(p[3]);
    g.paged_attention = reinterpret_cast<decltype(g.paged_attention)>(p[4]);
    g.copy_pages = reinterpret_cast<decltype(g.copy_pages)>(p[5]);
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction as_method(F f)
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"bind", as_method(native_bind), METH_FASTCALL, nullptr},
    {"rotary", as_method(native_rotary), METH_FASTCALL, nullptr},
    {"rotary_embedding", as_method(native_rotary_embedding), METH_FASTCALL, nullptr},
    {"cache_append", as_method(native_cache_append), METH_FASTCALL, nullptr},
    {"cache_gather", as_method(native_cache_gather), METH_FASTCALL, nullptr},
    {"attend", as_method(native_attend), METH_FASTCALL, nullptr},
    {"copy_pages", as_method(native_copy_pages), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
