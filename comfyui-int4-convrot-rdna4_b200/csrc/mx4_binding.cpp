// Python binding of the MX4 entries and of the operators around them (module _mx4_binding, used by
// _int4/mx4.py, _int4/rope.py and the W8A8 linear behind a norm):
// argument checks, output and workspace allocation on torch's caching allocator,
// and the launch on the device's current stream. A decode step calls these
// entries every few microseconds, and through ctypes and torch's Python calls the
// host took 9 to 20 us a call where the launch itself takes 3.
//
// Bad arguments raise ValueError, a refused or failed launch RuntimeError. No C++
// exception leaves an entry (HANDLE_TH_ERRORS).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <optional>

#include "convrot_b200.h"

namespace {

using at::Tensor;

constexpr int64_t kBlock = 32;

Tensor tensor(PyObject* o, const char* what) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, what, " must be an integer");
    }
    return v;
}

// dtype code of the C entries, -1 for another type.
int code_of(at::ScalarType t) {
    return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

int dtype_code(at::ScalarType t) {
    const int code = code_of(t);
    TORCH_CHECK_VALUE(code >= 0, "unsupported dtype ", t, ": float32, bfloat16 or float16");
    return code;
}

at::ScalarType dtype_arg(PyObject* o) {
    TORCH_CHECK_TYPE(THPDtype_Check(o), "dtype must be a torch.dtype");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

int group_of(int64_t k, PyObject* o) {
    const int64_t g = o == Py_None ? 0 : integer(o, "convrot_groupsize");
    TORCH_CHECK_VALUE(g == 0 || g == 16 || g == 64 || g == 256,
                      "convrot_groupsize must be 16, 64, 256 or 0 (not rotated), got ", g);
    TORCH_CHECK_VALUE(k > 0 && k % kBlock == 0, "MX4 needs a last dimension that is a positive multiple of 32, got ", k);
    TORCH_CHECK_VALUE(g == 0 || k % g == 0, "K=", k, " not divisible by convrot_groupsize ", g);
    return static_cast<int>(g);
}

int small(int64_t v, const char* what) {
    TORCH_CHECK_VALUE(v <= INT_MAX, what, " is too large: ", v);
    return static_cast<int>(v);
}

void on_device(const Tensor& t, const at::Device& d) {
    TORCH_CHECK_VALUE(t.is_cuda(), "the B200 ConvRot kernels need CUDA tensors");
    TORCH_CHECK_VALUE(t.device() == d, "tensors on ", d, " and ", t.device());
}

void* stream_of(const at::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

void check(const char* name, int rc) {
    if (rc == 0) return;
    TORCH_CHECK(rc != -1, name, " rejected its arguments: ", ck_convrot_last_error());
    TORCH_CHECK(false, name, " failed, cudaError=", rc);
}

// x [..., K] as a matrix whose rows are contiguous (a view where strides allow it).
Tensor rows_of(const Tensor& x) {
    Tensor m = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    if (m.stride(1) != 1 || (m.size(0) > 1 && m.stride(0) < m.size(1))) m = m.contiguous();
    return m;
}

at::DimVector with_last(const Tensor& x, int64_t last) {
    at::DimVector s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}

bool tiles_match(const Tensor& scales, int64_t rows, int64_t k) {
    return scales.dim() == 3 && scales.size(0) == (rows + 127) / 128 && scales.size(1) == (k + 127) / 128 && scales.size(2) == 512;
}

// (rows, K) of packed codes [..., K/2] and their tiled scales.
std::pair<int64_t, int64_t> codes_of(const Tensor& codes, const Tensor& scales, const char* what) {
    TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what, " codes and scales must be uint8");
    TORCH_CHECK_VALUE(codes.dim() >= 1 && codes.is_contiguous() && scales.is_contiguous(), what, " codes and scales must be contiguous");
    const int64_t k = codes.size(-1) * 2, rows = k ? codes.numel() / codes.size(-1) : 0;
    TORCH_CHECK_VALUE(tiles_match(scales, rows, k), what, " scales ", scales.sizes(), " do not match codes ", codes.sizes());
    return {rows, k};
}

PyObject* pair_of(Tensor a, Tensor b) {
    PyObject* t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

bool count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}

// quantize(x, group) -> (codes, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 2)) return nullptr;
    const Tensor x = tensor(a[0], "x");
    TORCH_CHECK_VALUE(x.dim() >= 1, "quantize_convrot_mx4 needs at least one dimension");
    const int64_t k = x.size(-1);
    const int group = group_of(k, a[1]), code = dtype_code(x.scalar_type());
    on_device(x, x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor m = rows_of(x);
    const int64_t rows = m.size(0);
    const auto bytes = m.options().dtype(at::kByte);
    Tensor codes = at::empty(with_last(x, k / 2), bytes);
    Tensor scales = at::empty({(rows + 127) / 128, (k + 127) / 128, 512}, bytes);
    check("ck_mx4_quant", ck_mx4_quant(m.const_data_ptr(), code, rows > 1 ? m.stride(0) : k, codes.data_ptr(), scales.data_ptr(),
                                       small(rows, "rows"), small(k, "K"), group, stream_of(x.device())));
    return pair_of(std::move(codes), std::move(scales));
    END_HANDLE_TH_ERRORS
}

// dequantize(codes, scales, group, dtype) -> values
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 4)) return nullptr;
    const Tensor codes = tensor(a[0], "codes"), scales = tensor(a[1], "scales");
    const auto [rows, k] = codes_of(codes, scales, "MX4");
    const int group = group_of(k, a[2]);
    const at::ScalarType type = dtype_arg(a[3]);
    const int code = dtype_code(type);
    on_device(codes, codes.device());
    on_device(scales, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    Tensor out = at::empty(with_last(codes, k), codes.options().dtype(type));
    check("ck_mx4_dequant", ck_mx4_dequant(codes.const_data_ptr(), scales.const_data_ptr(), out.data_ptr(), code, small(rows, "rows"),
                                           small(k, "K"), group, stream_of(codes.device())));
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// linear(x, qweight, wscales, bias or None, group) -> out
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 5)) return nullptr;
    const Tensor x = tensor(a[0], "x"), w = tensor(a[1], "qweight"), ws = tensor(a[2], "wscales");
    TORCH_CHECK_VALUE(w.dim() == 2, "qweight must be [N, K/2], got ", w.sizes());
    const auto [outs, k] = codes_of(w, ws, "weight");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "Input ", x.sizes(), " does not match qweight K=", k);
    const int group = group_of(k, a[4]), code = dtype_code(x.scalar_type());
    Tensor bias;
    int bias_code = 0;
    if (a[3] != Py_None) {
        bias = tensor(a[3], "bias");
        bias_code = code_of(bias.scalar_type());
        TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == outs && bias_code >= 0, "bias must be [", outs,
                          "] in float32, bfloat16 or float16");
    }
    on_device(x, x.device());
    on_device(w, x.device());
    on_device(ws, x.device());
    if (bias.defined()) {
        on_device(bias, x.device());
        bias = bias.contiguous();
    }
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor m = rows_of(x);
    const int rows = small(m.size(0), "rows"), cols = small(k, "K");
    Tensor out = at::empty(with_last(x, outs), m.options());
    const size_t need = ck_mx4_linear_workspace_size(rows, cols);
    Tensor workspace;
    if (need) workspace = at::empty({static_cast<int64_t>(need)}, m.options().dtype(at::kByte));
    check("ck_mx4_linear", ck_mx4_linear(m.const_data_ptr(), code, rows > 1 ? m.stride(0) : k, w.const_data_ptr(), ws.const_data_ptr(),
                                         bias.defined() ? bias.const_data_ptr() : nullptr, bias_code, out.data_ptr(), rows,
                                         small(outs, "N"), cols, group, need ? workspace.data_ptr() : nullptr, need, stream_of(x.device())));
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

struct Cache {
    int64_t pages;
    int heads, d, page, group;
};

Cache cache_of(const Tensor& codes, const Tensor& scales, PyObject* group) {
    TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, "cache codes and scales must be uint8");
    TORCH_CHECK_VALUE(codes.dim() == 5 && codes.size(1) == 2 && codes.is_contiguous() && scales.is_contiguous(),
                      "cache codes must be contiguous [pages, 2, heads, page, D/2]");
    const int64_t d = codes.size(4) * 2;
    TORCH_CHECK_VALUE(d == 64 || d == 128 || d == 256, "head_dim must be one of 64, 128, 256, got ", d);
    TORCH_CHECK_VALUE(scales.dim() == 5 && scales.size(0) == codes.size(0) && scales.size(1) == 2 && scales.size(2) == codes.size(2) &&
                          scales.size(3) == codes.size(3) && scales.size(4) == d / kBlock,
                      "cache scales ", scales.sizes(), " do not match codes ", codes.sizes());
    const int64_t page = codes.size(3);
    TORCH_CHECK_VALUE(page > 0 && page <= 65536 && (page & (page - 1)) == 0, "the page size must be a power of two up to 65536, got ", page);
    TORCH_CHECK_VALUE(codes.size(2) > 0, "the cache has no heads");
    return {codes.size(0), small(codes.size(2), "heads"), static_cast<int>(d), static_cast<int>(page), group_of(d, group)};
}

void check_slots(const Tensor& slots, int64_t t) {
    TORCH_CHECK_VALUE(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous() && (t < 0 || slots.size(0) == t),
                      "slots must be a contiguous int64 vector, one a token");
}

// cache_append(codes, scales, k, v, slots, group)
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 6)) return nullptr;
    const Tensor codes = tensor(a[0], "codes"), scales = tensor(a[1], "scales"), slots = tensor(a[4], "slots");
    Tensor k = tensor(a[2], "k"), v = tensor(a[3], "v");
    const Cache c = cache_of(codes, scales, a[5]);
    TORCH_CHECK_VALUE(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == c.heads && k.size(2) == c.d && k.scalar_type() == v.scalar_type(),
                      "keys ", k.sizes(), " and values ", v.sizes(), " must both be [T, ", c.heads, ", ", c.d, "] of one dtype");
    check_slots(slots, k.size(0));
    const int code = dtype_code(k.scalar_type());
    for (const Tensor* t : std::initializer_list<const Tensor*>{&codes, &scales, &k, &v, &slots}) on_device(*t, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    if (k.stride(2) != 1) k = k.contiguous();
    if (v.stride(2) != 1) v = v.contiguous();
    check("ck_mx4_cache_append",
          ck_mx4_cache_append(codes.data_ptr(), scales.data_ptr(), c.pages, c.heads, c.d, c.page, c.group, k.const_data_ptr(),
                              v.const_data_ptr(), code, k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.const_data_ptr(),
                              small(k.size(0), "tokens"), stream_of(codes.device())));
    // written in place: what autograd saved of them is out of date (inference tensors have no version)
    for (const Tensor* t : {&codes, &scales})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// cache_read(codes, scales, slots, dtype, group) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 5)) return nullptr;
    const Tensor codes = tensor(a[0], "codes"), scales = tensor(a[1], "scales"), slots = tensor(a[2], "slots");
    const Cache c = cache_of(codes, scales, a[4]);
    check_slots(slots, -1);
    const at::ScalarType type = dtype_arg(a[3]);
    const int code = dtype_code(type);
    for (const Tensor* t : {&codes, &scales, &slots}) on_device(*t, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    const int64_t t = slots.size(0);
    const auto options = codes.options().dtype(type);
    Tensor k = at::empty({t, c.heads, c.d}, options), v = at::empty({t, c.heads, c.d}, options);
    check("ck_mx4_cache_read",
          ck_mx4_cache_read(codes.const_data_ptr(), scales.const_data_ptr(), c.pages, c.heads, c.d, c.page, c.group,
                            slots.const_data_ptr(), small(t, "tokens"), k.data_ptr(), v.data_ptr(), code, stream_of(codes.device())));
    return pair_of(std::move(k), std::move(v));
    END_HANDLE_TH_ERRORS
}

Tensor queries_of(Tensor q, const Cache& c) {
    TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == c.d && q.size(1) > 0 && q.size(2) > 0 && c.heads > 0 && q.size(2) % c.heads == 0, "q ",
                      q.sizes(), " must be [B, Tq, a multiple of ", c.heads, ", ", c.d, "]");
    TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "queries must be bfloat16 or float16, got ",
                      q.scalar_type());
    return q;
}

void check_tables(const Tensor& table, const Tensor& lens, int64_t b) {
    TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == b && (table.size(1) <= 1 || table.stride(1) == 1) &&
                          (b <= 1 || table.stride(0) >= table.size(1)),
                      "block_table must be int32 [B, pages of a sequence] with contiguous rows");
    TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == b && lens.is_contiguous(),
                      "seq_lens must be a contiguous int32 vector [B]");
}

double scale_of(PyObject* o, const Cache& c) {
    if (o == Py_None) return 1.0 / std::sqrt(static_cast<double>(c.d));
    const double scale = PyFloat_AsDouble(o);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    return scale;
}

// attention(q, codes, scales, block_table, seq_lens, softmax_scale or None, group) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 7)) return nullptr;
    const Tensor codes = tensor(a[1], "codes"), scales = tensor(a[2], "scales"), table = tensor(a[3], "block_table"),
                 lens = tensor(a[4], "seq_lens");
    const Cache c = cache_of(codes, scales, a[6]);
    Tensor q = queries_of(tensor(a[0], "q"), c);
    const int64_t b = q.size(0);
    check_tables(table, lens, b);
    const double scale = scale_of(a[5], c);
    for (const Tensor* t : std::initializer_list<const Tensor*>{&q, &codes, &scales, &table, &lens}) on_device(*t, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    if (q.stride(3) != 1) q = q.contiguous();
    const int tq = small(q.size(1), "Tq"), hq = small(q.size(2), "Hq"), seqs = small(b, "B");
    const int64_t per = table.size(1);
    Tensor out = at::empty({b, tq, hq, c.d}, q.options());
    const size_t need = ck_mx4_attention_workspace_size(seqs, tq, hq, c.heads, c.d, per * c.page);
    Tensor workspace;
    if (need) workspace = at::empty({static_cast<int64_t>(need)}, codes.options());
    check("ck_mx4_attention",
          ck_mx4_attention(q.const_data_ptr(), code_of(q.scalar_type()), q.stride(0), q.stride(1), q.stride(2), codes.const_data_ptr(),
                           scales.const_data_ptr(), c.pages, c.page, table.const_data_ptr(), b > 1 ? table.stride(0) : per,
                           small(per, "pages of a sequence"), lens.const_data_ptr(), out.data_ptr(), seqs, tq, hq, c.heads, c.d, c.group,
                           static_cast<float>(scale), need ? workspace.data_ptr() : nullptr, need, stream_of(codes.device())));
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Positions, frequencies and sections of a rotary call on tokens of sizes `lead`.
struct Rope {
    Tensor positions, freqs;
    int type = 0, axes = 1, interleaved = 0;
    int sections[8] = {};
    // stride of the lead dimension `at` (its last: -1), 0 where there is none
    long long stride(int64_t at) const {
        const int64_t dims = positions.dim() - (axes > 1), i = dims + at;
        return i >= 0 ? positions.stride(i) : 0;
    }
    long long axis_stride() const { return axes > 1 ? positions.stride(positions.dim() - 1) : 0; }
};

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, "expected a truth value");
    }
    return v != 0;
}

Rope rope_of(at::IntArrayRef lead, int64_t d, PyObject* positions, PyObject* freqs, PyObject* sections, PyObject* interleaved) {
    Rope r;
    r.positions = tensor(positions, "positions");
    r.freqs = tensor(freqs, "freqs");
    TORCH_CHECK_VALUE(d > 0 && d % 2 == 0, "rotary positions need an even head dimension, got ", d);
    TORCH_CHECK_VALUE(r.freqs.scalar_type() == at::kDouble && r.freqs.dim() == 1, "freqs must be float64 [pairs]");
    const int64_t pairs = r.freqs.size(0);
    TORCH_CHECK_VALUE(2 * pairs <= d, pairs, " pairs do not fit a head of ", d);
    if (sections == Py_None) {
        r.sections[0] = static_cast<int>(pairs);
    } else {
        TORCH_CHECK_TYPE(PyTuple_Check(sections) || PyList_Check(sections), "sections must be a tuple or a list of integers");
        const Py_ssize_t n = PySequence_Size(sections);
        TORCH_CHECK_VALUE(n >= 1 && n <= 8, "sections must name 1 to 8 axes, got ", n);
        int64_t sum = 0;
        for (Py_ssize_t i = 0; i < n; ++i) {
            const int64_t v = integer(PyTuple_Check(sections) ? PyTuple_GET_ITEM(sections, i) : PyList_GET_ITEM(sections, i), "a section");
            TORCH_CHECK_VALUE(v >= 0 && v <= pairs, "sections must add up to the ", pairs, " pairs of freqs");
            sum += v;
            r.sections[i] = static_cast<int>(v);
        }
        TORCH_CHECK_VALUE(sum == pairs, "sections must add up to the ", pairs, " pairs of freqs");
        r.axes = static_cast<int>(n);
    }
    const at::ScalarType t = r.positions.scalar_type();
    TORCH_CHECK_VALUE(t == at::kInt || t == at::kLong || t == at::kFloat, "positions must be int32, int64 or float32, got ", t);
    r.type = t == at::kInt ? 0 : t == at::kLong ? 1 : 2;
    r.interleaved = truth(interleaved);
    at::DimVector want(lead.begin(), lead.end());
    if (r.axes > 1) want.push_back(r.axes);
    if (r.positions.sizes() != at::IntArrayRef(want)) {
        bool fits = r.positions.dim() <= static_cast<int64_t>(want.size());
        for (int64_t i = 1; fits && i <= r.positions.dim(); ++i)
            fits = r.positions.size(-i) == want[want.size() - i] || (r.positions.size(-i) == 1 && !(r.axes > 1 && i == 1));
        TORCH_CHECK_VALUE(fits, "positions ", r.positions.sizes(), " do not fit tokens ", lead, " on ", r.axes, r.axes > 1 ? " axes" : " axis");
        r.positions = r.positions.expand(want);
    }
    return r;
}

// rope(x, positions, freqs, sections or None, interleaved, inverse) -> out
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 6)) return nullptr;
    Tensor x = tensor(a[0], "x");
    TORCH_CHECK_VALUE(x.dim() >= 2, "x must be [..., heads, D], got ", x.sizes());
    const int64_t heads = x.size(-2), d = x.size(-1);
    const int code = dtype_code(x.scalar_type());
    Rope r = rope_of(x.sizes().slice(0, x.dim() - 2), d, a[1], a[2], a[3], a[4]);
    const bool inverse = truth(a[5]);
    for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &r.positions, &r.freqs}) on_device(*t, x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor out = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (x.dim() > 4) {                                            // [B, T, heads, D], by a copy where strides do not allow a view
        const int64_t t = x.size(-3);
        int64_t b = 1;
        for (int64_t i = 0; i < x.dim() - 3; ++i) b *= x.size(i);
        r.positions = r.positions.reshape(r.axes > 1 ? at::DimVector{b, t, r.axes} : at::DimVector{b, t});
        x = x.reshape({b, t, heads, d});
    }
    if (x.stride(-1) != 1) x = x.contiguous();
    r.freqs = r.freqs.contiguous();
    const bool has_t = x.dim() >= 3, has_b = x.dim() == 4;
    check("ck_rope", ck_rope(x.const_data_ptr(), code, has_b ? x.stride(0) : 0, has_t ? x.stride(-3) : 0, x.stride(-2), out.data_ptr(),
                             has_b ? small(x.size(0), "batch") : 1, has_t ? small(x.size(-3), "tokens") : 1, small(heads, "heads"), small(d, "D"),
                             r.positions.const_data_ptr(), r.type, has_b ? r.stride(-2) : 0, has_t ? r.stride(-1) : 0, r.axis_stride(),
                             r.freqs.const_data_ptr(), r.sections, r.axes, r.interleaved, inverse, stream_of(x.device())));
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// cache_append_rope(codes, scales, q or None, k, v, slots, positions, freqs, sections or None, interleaved, group) -> q or None
PyObject* cache_append_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 11)) return nullptr;
    const Tensor codes = tensor(a[0], "codes"), scales = tensor(a[1], "scales"), slots = tensor(a[5], "slots");
    Tensor k = tensor(a[3], "k"), v = tensor(a[4], "v"), q;
    const Cache c = cache_of(codes, scales, a[10]);
    TORCH_CHECK_VALUE(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == c.heads && k.size(2) == c.d && k.scalar_type() == v.scalar_type(),
                      "keys ", k.sizes(), " and values ", v.sizes(), " must both be [T, ", c.heads, ", ", c.d, "] of one dtype");
    const int64_t t = k.size(0);
    check_slots(slots, t);
    const int code = dtype_code(k.scalar_type());
    if (a[2] != Py_None) {
        q = tensor(a[2], "q");
        TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == t && q.size(2) == c.d && q.scalar_type() == k.scalar_type(), "queries ", q.sizes(),
                          " must be [", t, ", heads, ", c.d, "] in the keys' dtype");
    }
    Rope r = rope_of(k.sizes().slice(0, 1), c.d, a[6], a[7], a[8], a[9]);
    for (const Tensor* x : std::initializer_list<const Tensor*>{&codes, &scales, &k, &v, &slots, &r.positions, &r.freqs}) on_device(*x, codes.device());
    if (q.defined()) on_device(q, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    if (k.stride(2) != 1) k = k.contiguous();
    if (v.stride(2) != 1) v = v.contiguous();
    if (q.defined() && q.stride(2) != 1) q = q.contiguous();
    r.freqs = r.freqs.contiguous();
    Tensor out;
    if (q.defined()) out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    check("ck_mx4_cache_append_rope",
          ck_mx4_cache_append_rope(codes.data_ptr(), scales.data_ptr(), c.pages, c.heads, c.d, c.page, c.group,
                                   q.defined() ? q.const_data_ptr() : nullptr, k.const_data_ptr(), v.const_data_ptr(), code,
                                   q.defined() ? small(q.size(1), "query heads") : 0, q.defined() ? q.stride(0) : 0, q.defined() ? q.stride(1) : 0,
                                   k.stride(0), k.stride(1), v.stride(0), v.stride(1), q.defined() ? out.data_ptr() : nullptr,
                                   slots.const_data_ptr(), small(t, "tokens"), r.positions.const_data_ptr(), r.type, r.stride(-1), r.axis_stride(),
                                   r.freqs.const_data_ptr(), r.sections, r.axes, r.interleaved, stream_of(codes.device())));
    for (const Tensor* x : {&codes, &scales})                     // (as cache_append)
        if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
    if (!q.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// tree_attention(q, codes, scales, block_table, seq_lens, tree_mask, tree_lens or None, softmax_scale or None, group) -> out
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 9)) return nullptr;
    const Tensor codes = tensor(a[1], "codes"), scales = tensor(a[2], "scales"), table = tensor(a[3], "block_table"),
                 lens = tensor(a[4], "seq_lens");
    const Cache c = cache_of(codes, scales, a[8]);
    Tensor q = queries_of(tensor(a[0], "q"), c);
    const int64_t b = q.size(0), t = q.size(1);
    check_tables(table, lens, b);
    Tensor mask = tensor(a[5], "tree_mask"), nodes;
    TORCH_CHECK_VALUE(mask.scalar_type() == at::kBool, "tree_mask must be bool, got ", mask.scalar_type());
    TORCH_CHECK_VALUE((mask.dim() == 2 || (mask.dim() == 3 && mask.size(0) == b)) && mask.size(-1) == t && mask.size(-2) == t, "tree_mask ",
                      mask.sizes(), " must be [", t, ", ", t, "] or [", b, ", ", t, ", ", t, "]");
    if (a[6] != Py_None) {
        nodes = tensor(a[6], "tree_lens");
        TORCH_CHECK_VALUE(nodes.scalar_type() == at::kInt && nodes.dim() == 1 && nodes.size(0) == b && nodes.is_contiguous(),
                          "tree_lens must be a contiguous int32 vector [B]");
    }
    const double scale = scale_of(a[7], c);
    for (const Tensor* x : std::initializer_list<const Tensor*>{&q, &codes, &scales, &table, &lens, &mask}) on_device(*x, codes.device());
    if (nodes.defined()) on_device(nodes, codes.device());
    const c10::cuda::CUDAGuard guard(codes.device());
    if (q.stride(3) != 1) q = q.contiguous();
    if (mask.stride(-1) != 1 && t > 1) mask = mask.contiguous();
    const int tq = small(t, "T"), hq = small(q.size(2), "Hq"), seqs = small(b, "B");
    const int64_t per = table.size(1);
    Tensor out = at::empty({b, tq, hq, c.d}, q.options());
    const size_t need = ck_mx4_tree_attention_workspace_size(seqs, tq, hq, c.heads, c.d, per * c.page);
    Tensor workspace;
    if (need) workspace = at::empty({static_cast<int64_t>(need)}, codes.options());
    check("ck_mx4_tree_attention",
          ck_mx4_tree_attention(q.const_data_ptr(), code_of(q.scalar_type()), q.stride(0), q.stride(1), q.stride(2), codes.const_data_ptr(),
                                scales.const_data_ptr(), c.pages, c.page, table.const_data_ptr(), b > 1 ? table.stride(0) : per,
                                small(per, "pages of a sequence"), lens.const_data_ptr(), nodes.defined() ? nodes.const_data_ptr() : nullptr,
                                mask.const_data_ptr(), mask.dim() == 3 ? mask.stride(0) : 0, mask.stride(-2), out.data_ptr(), seqs, tq, hq,
                                c.heads, c.d, c.group, static_cast<float>(scale), need ? workspace.data_ptr() : nullptr, need,
                                stream_of(codes.device())));
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// linear_rmsnorm(x, qweight, wscales, bias or None, norm_weight or None, residual or None, eps, group) -> (out, hidden)
PyObject* linear_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!count(n, 8)) return nullptr;
    const Tensor x = tensor(a[0], "x");
    Tensor w = tensor(a[1], "qweight"), ws = tensor(a[2], "wscales"), bias, gain, residual;
    TORCH_CHECK_VALUE(w.dim() == 2 && w.scalar_type() == at::kChar, "qweight must be int8 [N, K], got ", w.sizes());
    const int64_t outs = w.size(0), k = w.size(1), group = integer(a[7], "convrot_groupsize");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "Input ", x.sizes(), " does not match qweight K=", k);
    TORCH_CHECK_VALUE(group == 16 || group == 64 || group == 256, "convrot_groupsize must be 16, 64 or 256, got ", group);
    TORCH_CHECK_VALUE(k > 0 && k % group == 0, "Input K=", k, " not divisible by convrot_groupsize ", group);
    TORCH_CHECK_VALUE(k <= 16384, "Input K=", k, " is larger than 16384");
    TORCH_CHECK_VALUE(ws.numel() == outs, "wscales must hold a scale for each of the ", outs, " outputs, got ", ws.sizes());
    const int code = dtype_code(x.scalar_type());
    const double eps = PyFloat_AsDouble(a[6]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    auto vector = [&](PyObject* o, const char* what, int64_t size) {
        Tensor v;
        if (o == Py_None) return v;
        v = tensor(o, what);
        TORCH_CHECK_VALUE(v.dim() == 1 && v.size(0) == size && code_of(v.scalar_type()) >= 0, what, " must be [", size,
                          "] in float32, bfloat16 or float16");
        return v;
    };
    bias = vector(a[3], "bias", outs);
    gain = vector(a[4], "norm_weight", k);
    if (a[5] != Py_None) {
        residual = tensor(a[5], "residual");
        TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), "residual ", residual.sizes(),
                          " must have the shape and dtype of x ", x.sizes());
    }
    for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &w, &ws, &bias, &gain, &residual})
        if (t->defined()) on_device(*t, x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor m = rows_of(x);
    w = w.contiguous();
    ws = ws.to(at::kFloat).contiguous();
    if (bias.defined()) bias = bias.contiguous();
    if (gain.defined()) gain = gain.contiguous();
    Tensor r, hidden = x;
    if (residual.defined()) {
        r = rows_of(residual);
        hidden = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    }
    const int rows = small(m.size(0), "rows"), cols = small(k, "K");
    // (the product's epilogue writes fp32 or bf16)
    const at::ScalarType type = x.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
    Tensor out = at::empty(with_last(x, outs), m.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
    const size_t need = ck_convrot_w8a8_linear_rmsnorm_workspace_size(rows, cols);
    Tensor workspace;
    if (need) workspace = at::empty({static_cast<int64_t>(need)}, m.options().dtype(at::kByte));
    check("ck_convrot_w8a8_linear_rmsnorm",
          ck_convrot_w8a8_linear_rmsnorm(m.const_data_ptr(), r.defined() ? r.const_data_ptr() : nullptr, code, rows > 1 ? m.stride(0) : k,
                                         r.defined() && rows > 1 ? r.stride(0) : k, gain.defined() ? gain.const_data_ptr() : nullptr,
                                         gain.defined() ? code_of(gain.scalar_type()) : 0, static_cast<float>(eps), w.const_data_ptr(),
                                         ws.const_data_ptr(), bias.defined() ? bias.const_data_ptr() : nullptr,
                                         bias.defined() ? code_of(bias.scalar_type()) : 0, r.defined() ? hidden.data_ptr() : nullptr,
                                         out.data_ptr(), type == at::kBFloat16, rows, small(outs, "N"), cols, static_cast<int>(group),
                                         need ? workspace.data_ptr() : nullptr, need, stream_of(x.device())));
    return pair_of(out.to(x.scalar_type()), std::move(hidden));
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef methods[] = {
    {"quantize", fast<quantize>(), METH_FASTCALL, nullptr},         {"dequantize", fast<dequantize>(), METH_FASTCALL, nullptr},
    {"linear", fast<linear>(), METH_FASTCALL, nullptr},             {"cache_append", fast<cache_append>(), METH_FASTCALL, nullptr},
    {"cache_read", fast<cache_read>(), METH_FASTCALL, nullptr},     {"attention", fast<attention>(), METH_FASTCALL, nullptr},
    {"rope", fast<rope>(), METH_FASTCALL, nullptr},                 {"cache_append_rope", fast<cache_append_rope>(), METH_FASTCALL, nullptr},
    {"tree_attention", fast<tree_attention>(), METH_FASTCALL, nullptr}, {"linear_rmsnorm", fast<linear_rmsnorm>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mx4_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mx4_binding() { return PyModule_Create(&module); }
