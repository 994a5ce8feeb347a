// Python entry points of the paged key-value cache: argument checks, output tensors, the argument blocks of the
// C ABI and the current stream, in one native call.  A decode step of a short sequence takes a few microseconds on the
// GPU; the same checks and allocations written in Python take 9 to 17 and would set the step's time.
//
// The module is `_paged_binding`; the functions with names, defaults and documentation are in paged.py and
// pass everything on by position.
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <limits>
#include <optional>
#include <string>

#include "../../include/anchor_attn_b200.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kMaxNewTokens = 16;     // tokens of one sequence a decode call takes

// A refused argument: AssertionError in Python.
struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};

std::string text(const char* s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
template <typename... A>
[[noreturn]] __attribute__((noinline, cold)) void refuse(const A&... parts) {
    std::string s;
    ((s += text(parts)), ...);
    throw Refused(s);
}
#define REQUIRE(ok, ...)                          \
    do {                                          \
        if (__builtin_expect(!(ok), 0)) refuse(__VA_ARGS__); \
    } while (0)

PyObject* g_status_words = nullptr;       // {device index: int32 tensor}
PyObject* g_new_status_word = nullptr;    // makes one

const at::Tensor& tensor(PyObject* o, const char* name) {
    REQUIRE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
// None: an undefined tensor
const at::Tensor& optional_tensor(PyObject* o, const char* name) {
    static const at::Tensor none;
    return o == Py_None ? none : tensor(o, name);
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v == 1;
}
int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

template <typename T = void>
T* data(const at::Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

void need_int32(const at::Tensor& t, const char* name, int64_t dim, const at::Device& device) {
    REQUIRE(t.scalar_type() == at::kInt && t.dim() == dim && t.device() == device, name, " must be a ", dim,
            "-dimensional int32 tensor on the device of the inputs");
}
// bf16 whose last axis is a row of 128 values
void need_rows(const at::Tensor& t, const char* name, const at::Device& device) {
    REQUIRE(t.scalar_type() == at::kBFloat16 && t.device() == device, name,
            " must be bfloat16 on the device of the other tensors");
    REQUIRE(t.dim() >= 1 && t.size(-1) == kHeadDim, "head dimension ", t.dim() ? t.size(-1) : 0, " is not supported (128 only)");
}
// contiguous rows, strides and address of 16-byte multiples: what the kernels read in place
bool usable(const at::Tensor& t) {
    const auto st = t.strides();
    bool ok = st.back() == 1 && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
    for (size_t i = 0; i + 1 < st.size(); ++i) ok = ok && !(st[i] & 7);
    return ok;
}
// an expanded view, whose indices share memory: no place to write to
bool shares_memory(const at::Tensor& t) { return at::has_internal_overlap(t) == at::MemOverlap::Yes; }
at::Tensor in_place_or_copy(const at::Tensor& t) { return usable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

bool page_size_ok(int64_t n) { return n >= 16 && n <= 256 && !(n & (n - 1)); }
int32_t int32_of(int64_t v, const char* name) {
    REQUIRE(v >= 0 && v <= INT32_MAX, name, " ", v, " is out of range");
    return (int32_t)v;
}

void fill_table(aa_paged_cache_t& c, const at::Tensor& table, const at::Tensor& lens, const at::Device& device) {
    need_int32(table, "block_table", 2, device);
    need_int32(lens, "seq_lens", 1, device);
    c.B = int32_of(table.size(0), "batch");
    c.table_width = int32_of(table.size(1), "table width");
    REQUIRE(lens.size(0) == c.B && (c.B < 2 || lens.stride(0) == 1), "seq_lens must be a contiguous [B] tensor");
    REQUIRE(c.table_width >= 1 && (c.table_width == 1 || table.stride(1) == 1), "the rows of block_table must be contiguous");
    c.block_table = data<int32_t>(table);
    c.table_stride = table.stride(0);
    c.seq_lens = data<int32_t>(lens);
    c.D = kHeadDim;
}

void need_scale(const at::Tensor& t, const char* name, int64_t heads, const at::Device& device) {
    REQUIRE(t.defined() && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == heads && t.device() == device &&
                t.is_contiguous(),
            name, " must be a contiguous fp32 [Hkv] tensor: the pools are float8_e4m3fn");
}

aa_paged_cache_t make_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                            const at::Tensor& k_scale, const at::Tensor& v_scale) {
    aa_paged_cache_t c{};
    const at::Device device = k.device();
    REQUIRE(k.dim() == 4 && v.sizes() == k.sizes() && k.size(3) == kHeadDim,
            "k_pages and v_pages must both be [pages, Hkv, page_size, 128]");
    const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
    REQUIRE((fp8 || k.scalar_type() == at::kBFloat16) && v.scalar_type() == k.scalar_type() && v.device() == device,
            "k_pages and v_pages must both be bfloat16 or both float8_e4m3fn, on one device");
    REQUIRE(page_size_ok(k.size(2)), "page size ", k.size(2), " is not a power of two from 16 to 256");
    const auto ks = k.strides(), vs = v.strides();
    const int64_t unit = fp8 ? 15 : 7;
    REQUIRE(ks[3] == 1 && vs[3] == 1, "the rows of the pools must be contiguous");
    REQUIRE(!((ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & unit) &&
                !((reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) & 15),
            "the rows of the pools must start on 16-byte boundaries");
    if (fp8) {
        need_scale(k_scale, "k_scale", k.size(1), device);
        need_scale(v_scale, "v_scale", k.size(1), device);
        c.k_scale = data<float>(k_scale);
        c.v_scale = data<float>(v_scale);
    } else {
        REQUIRE(!k_scale.defined() && !v_scale.defined(), "k_scale and v_scale belong to float8_e4m3fn pools");
    }
    fill_table(c, table, lens, device);
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    c.k_stride_page = ks[0]; c.k_stride_head = ks[1]; c.k_stride_row = ks[2];
    c.v_stride_page = vs[0]; c.v_stride_head = vs[1]; c.v_stride_row = vs[2];
    c.pages = int32_of(k.size(0), "number of pages");
    c.page_size = (int32_t)k.size(2);
    c.Hkv = int32_of(k.size(1), "KV heads");
    c.cache_dtype = fp8 ? AA_E4M3 : AA_BF16;
    return c;
}

// The device's status word.  The checks that need no GPU come before it.
uint32_t* status_word(const at::Device& device) {
    REQUIRE(device.is_cuda(), "the tensors of a paged cache must be CUDA tensors (there is no CPU path)");
    THPObjectPtr key(PyLong_FromLong(device.index()));
    if (!key) throw python_error();
    PyObject* word = PyDict_GetItemWithError(g_status_words, key.get());
    if (word) return static_cast<uint32_t*>(THPVariable_Unpack(word).data_ptr());
    if (PyErr_Occurred()) throw python_error();
    THPObjectPtr made(PyObject_CallFunctionObjArgs(g_new_status_word, key.get(), nullptr));
    if (!made) throw python_error();
    return static_cast<uint32_t*>(THPVariable_Unpack(made.get()).data_ptr());
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& device) {
    return at::Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

void raise_on(int rc, const char* what) {
    if (rc == AA_OK) return;
    std::string message = std::string(what) + ": " + aa_strerror(rc);
    if (rc == AA_ERR_CUDA) message += std::string(": ") + aa_last_cuda_error();
    throw std::runtime_error(message);
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    THPObjectPtr x(a.defined() ? THPVariable_Wrap(a) : Py_NewRef(Py_None));
    THPObjectPtr y(b.defined() ? THPVariable_Wrap(b) : Py_NewRef(Py_None));
    return PyTuple_Pack(2, x.get(), y.get());
}

// Runs f, turning C++ exceptions into Python's.
template <typename F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_AssertionError, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

void need_codes(const at::Tensor& codes, const at::Tensor& scales, int64_t heads, const at::Device& device) {
    REQUIRE(codes.scalar_type() == at::kChar && codes.dim() == 3 && codes.size(1) == heads && codes.size(2) == kHeadDim &&
                codes.is_contiguous() && codes.device() == device,
            "key_codes must be a contiguous int8 [pages, Hkv, 128] tensor");
    REQUIRE(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == codes.size(0) &&
                scales.size(1) == heads && scales.is_contiguous() && scales.device() == device,
            "key_code_scales must be a contiguous fp32 [pages, Hkv] tensor");
}

// query [B, H, 128] or [B, new, H, 128]: its strides (sequence, token, head), new tokens and heads
struct Queries {
    at::Tensor t;
    int64_t sb, sn, sh;
    int32_t fresh, heads;
};
Queries make_queries(const at::Tensor& query, int64_t kv_heads, int64_t batch) {
    const bool flat = query.dim() == 3;
    REQUIRE((flat || query.dim() == 4) && query.size(0) == batch, "query must be [B, H, 128] or [B, new tokens, H, 128]");
    const int64_t fresh = flat ? 1 : query.size(1), heads = query.size(flat ? 1 : 2);
    REQUIRE(fresh >= 1 && fresh <= kMaxNewTokens, fresh, " new tokens: 1 to ", kMaxNewTokens,
            " are supported (dense_causal_attention takes longer chunks)");
    REQUIRE(kv_heads > 0 && heads % kv_heads == 0 && heads > 0, kv_heads, " KV heads do not divide ", heads, " query heads");
    Queries q{query, 0, 0, 0, (int32_t)fresh, int32_of(heads, "query heads")};
    return q;
}
void place(Queries& q) {
    q.t = in_place_or_copy(q.t);
    const auto st = q.t.strides();
    q.sb = st[0];
    q.sn = st.size() == 3 ? 0 : st[1];
    q.sh = st[st.size() - 2];
}

// (key, value, k_pages, v_pages, block_table, seq_lens, cu_seqlens, query, cos, sin, k_scale, v_scale, key_codes,
//  key_code_scales, return_key)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        REQUIRE(n == 15, "15 arguments expected");
        const at::Tensor &key = tensor(args[0], "key"), &value = tensor(args[1], "value"), &k = tensor(args[2], "k_pages"),
                         &v = tensor(args[3], "v_pages"), &cu = optional_tensor(args[6], "cu_seqlens"),
                         &query = optional_tensor(args[7], "query"), &cos = optional_tensor(args[8], "cos"),
                         &sin = optional_tensor(args[9], "sin"), &codes = optional_tensor(args[12], "key_codes"),
                         &scales = optional_tensor(args[13], "key_code_scales");
        const bool return_key = truth(args[14]);
        const at::Device device = k.device();
        aa_paged_append_t a{};
        a.cache = make_cache(k, v, tensor(args[4], "block_table"), tensor(args[5], "seq_lens"),
                             optional_tensor(args[10], "k_scale"), optional_tensor(args[11], "v_scale"));
        aa_paged_cache_t& c = a.cache;
        REQUIRE(!shares_memory(k) && !shares_memory(v), "pages of the pools share memory: they cannot be appended to");
        need_rows(key, "key", device);
        need_rows(value, "value", device);
        REQUIRE(key.dim() == 3 && value.sizes() == key.sizes() && key.size(1) == c.Hkv,
                "key and value must be [T, Hkv, 128] with the KV heads of the pools");
        a.T = int32_of(key.size(0), "tokens");
        if (cu.defined()) {
            need_int32(cu, "cu_seqlens", 1, device);
            REQUIRE(cu.size(0) == (int64_t)c.B + 1 && cu.stride(0) == 1, "cu_seqlens must be a contiguous [B + 1] tensor");
            a.cu_seqlens = data<int32_t>(cu);
        } else {
            REQUIRE(c.B == 0 || a.T % c.B == 0, a.T, " tokens do not divide among ", c.B, " sequences: pass cu_seqlens");
        }
        REQUIRE(cos.defined() == sin.defined(), "cos and sin go together");
        if (cos.defined()) {
            for (const at::Tensor* t : {&cos, &sin})
                REQUIRE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == kHeadDim / 2 && t->is_contiguous() &&
                            t->device() == device && !(reinterpret_cast<uintptr_t>(t->data_ptr()) & 15),
                        "cos and sin must be contiguous fp32 [positions, 64] tensors");
            a.cos = data<float>(cos);
            a.sin = data<float>(sin);
            a.rope_rows = int32_of(std::min(cos.size(0), sin.size(0)), "rotary positions");
        }
        REQUIRE(codes.defined() == scales.defined(), "key_codes and key_code_scales go together");
        if (codes.defined()) {
            need_codes(codes, scales, c.Hkv, device);
            REQUIRE(codes.size(0) == c.pages, "key_codes must have a row for every page of the pools");
            a.key_codes = data<int8_t>(codes);
            a.key_code_scales = data<float>(scales);
        }
        if (query.defined()) {
            need_rows(query, "query", device);
            REQUIRE(query.dim() == 3 && query.size(0) == a.T && query.size(1) > 0 && c.Hkv > 0 && query.size(1) % c.Hkv == 0,
                    "query must be [T, H, 128] with a multiple of the KV heads");
            a.H = int32_of(query.size(1), "query heads");
        }
        c.status = status_word(device);
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor query_out, key_out;
        if (query.defined()) query_out = empty({a.T, a.H, kHeadDim}, at::kBFloat16, device);
        if (return_key) key_out = empty({a.T, c.Hkv, kHeadDim}, at::kBFloat16, device);
        if (a.T == 0 || c.B == 0) return pair(query_out, key_out);
        const at::Tensor key_in = in_place_or_copy(key), value_in = in_place_or_copy(value);
        const at::Tensor query_in = query.defined() ? in_place_or_copy(query) : query;
        a.key = key_in.data_ptr();
        a.value = value_in.data_ptr();
        a.key_stride_t = key_in.stride(0); a.key_stride_h = key_in.stride(1);
        a.value_stride_t = value_in.stride(0); a.value_stride_h = value_in.stride(1);
        if (query.defined()) {
            a.query = query_in.data_ptr();
            a.query_out = query_out.data_ptr();
            a.query_stride_t = query_in.stride(0); a.query_stride_h = query_in.stride(1);
            a.query_out_stride_t = a.H * kHeadDim; a.query_out_stride_h = kHeadDim;
        }
        if (return_key) {
            a.key_out = key_out.data_ptr();
            a.key_out_stride_t = c.Hkv * kHeadDim; a.key_out_stride_h = kHeadDim;
        }
        raise_on(aa_paged_append(&a, c10::cuda::getCurrentCUDAStream(device.index()).stream()), "paged_kv_append");
        return pair(query_out, key_out);
    });
}

// (query, k_pages, v_pages, block_table, seq_lens, scaling, k_scale, v_scale, pages, page_counts, out, return_lse)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        REQUIRE(n == 12, "12 arguments expected");
        const at::Tensor &query = tensor(args[0], "query"), &k = tensor(args[1], "k_pages"), &v = tensor(args[2], "v_pages"),
                         &pages = optional_tensor(args[8], "pages"), &counts = optional_tensor(args[9], "page_counts"),
                         &out_in = optional_tensor(args[10], "out");
        const bool return_lse = truth(args[11]);
        const at::Device device = k.device();
        aa_paged_attend_t a{};
        a.cache = make_cache(k, v, tensor(args[3], "block_table"), tensor(args[4], "seq_lens"),
                             optional_tensor(args[6], "k_scale"), optional_tensor(args[7], "v_scale"));
        aa_paged_cache_t& c = a.cache;
        if (args[5] != Py_None) {
            a.sm_scale = PyFloat_AsDouble(args[5]);
            if (PyErr_Occurred()) throw python_error();
            // 0 stands for the default in the argument block; the smallest double is a scale of 0 in 32 bits
            if (a.sm_scale == 0.0) a.sm_scale = std::numeric_limits<double>::denorm_min();
        }
        need_rows(query, "query", device);
        Queries q = make_queries(query, c.Hkv, c.B);
        REQUIRE(pages.defined() == counts.defined(), "pages and page_counts go together");
        if (pages.defined()) {
            need_int32(pages, "pages", 3, device);
            need_int32(counts, "page_counts", 2, device);
            REQUIRE(pages.size(0) == c.B && pages.size(1) == c.Hkv && pages.size(2) >= 1 && pages.is_contiguous(),
                    "pages must be a contiguous [B, Hkv, width] tensor");
            REQUIRE(counts.size(0) == c.B && counts.size(1) == c.Hkv && counts.is_contiguous(),
                    "page_counts must be a contiguous [B, Hkv] tensor");
            a.pages = data<int32_t>(pages);
            a.page_counts = data<int32_t>(counts);
            a.list_width = int32_of(pages.size(2), "list width");
        }
        if (out_in.defined()) {
            need_rows(out_in, "out", device);
            REQUIRE(out_in.sizes() == query.sizes() && usable(out_in),
                    "out must have the shape of query, contiguous rows and strides and address of 16-byte multiples");
            REQUIRE(!shares_memory(out_in), "rows of out share memory");
            // rows are written while others are read
            REQUIRE(at::get_overlap_status(out_in, query) != at::MemOverlapStatus::Partial,
                    "out must be query itself or not overlap it");
        }
        c.status = status_word(device);
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor out = out_in.defined() ? out_in : empty(query.sizes(), at::kBFloat16, device);
        at::Tensor lse;
        if (return_lse) lse = empty(query.sizes().slice(0, query.dim() - 1), at::kFloat, device);
        if (c.B > 0) {
            place(q);
            a.q = q.t.data_ptr();
            a.q_stride_b = q.sb; a.q_stride_n = q.sn; a.q_stride_h = q.sh;
            const auto st = out.strides();
            a.out = out.data_ptr();
            a.o_stride_b = st[0];
            a.o_stride_n = st.size() == 3 ? 0 : st[1];
            a.o_stride_h = st[st.size() - 2];
            a.lse = data<float>(lse);
            a.Nq = q.fresh;
            a.H = q.heads;
            // The workspace is this call's own (the allocator hands it out again in stream order): calls on other
            // streams, and graphs captured from different calls, never meet in one.
            raise_on(aa_paged_attend_workspace_bytes(&a, &a.workspace_bytes), "paged_decode_attention");
            const at::Tensor workspace = empty({(int64_t)a.workspace_bytes}, at::kByte, device);
            a.workspace = workspace.data_ptr();
            raise_on(aa_paged_attend(&a, c10::cuda::getCurrentCUDAStream(device.index()).stream()), "paged_decode_attention");
        }
        if (!return_lse) return out_in.defined() ? Py_NewRef(args[10]) : THPVariable_Wrap(out);
        THPObjectPtr first(out_in.defined() ? Py_NewRef(args[10]) : THPVariable_Wrap(out));
        THPObjectPtr second(THPVariable_Wrap(lse));
        return PyTuple_Pack(2, first.get(), second.get());
    });
}

// (query, key_codes, key_code_scales, block_table, seq_lens, top_k, page_size, keep_first, keep_last)
PyObject* select(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        REQUIRE(n == 9, "9 arguments expected");
        const at::Tensor &query = tensor(args[0], "query"), &codes = tensor(args[1], "key_codes"),
                         &scales = tensor(args[2], "key_code_scales");
        const int64_t top = integer(args[5]), page = integer(args[6]), keep_first = integer(args[7]), keep_last = integer(args[8]);
        const at::Device device = query.device();
        need_rows(query, "query", device);
        REQUIRE(codes.dim() == 3, "key_codes must be a contiguous int8 [pages, Hkv, 128] tensor");
        need_codes(codes, scales, codes.size(1), device);
        aa_page_select_t a{};
        aa_paged_cache_t& c = a.cache;
        fill_table(c, tensor(args[3], "block_table"), tensor(args[4], "seq_lens"), device);
        c.Hkv = int32_of(codes.size(1), "KV heads");
        c.pages = int32_of(codes.size(0), "number of pages");
        Queries q = make_queries(query, c.Hkv, c.B);
        REQUIRE(page_size_ok(page), "page size ", page, " is not a power of two from 16 to 256");
        REQUIRE(keep_first >= 0 && keep_last >= 1 && keep_first <= top && keep_last <= top - keep_first,
                "keep_first must be at least 0, keep_last at least 1, and top_k hold both");
        c.page_size = (int32_t)page;
        a.top = int32_of(top, "top_k");
        a.keep_first = (int32_t)keep_first;
        a.keep_last = (int32_t)keep_last;
        c.status = status_word(device);
        const c10::cuda::OptionalCUDAGuard guard(device);
        at::Tensor lists = empty({c.B, c.Hkv, top}, at::kInt, device), counts = empty({c.B, c.Hkv}, at::kInt, device);
        if (c.B > 0) {
            place(q);
            a.q = q.t.data_ptr();
            a.q_stride_b = q.sb; a.q_stride_n = q.sn; a.q_stride_h = q.sh;
            a.key_codes = data<int8_t>(codes);
            a.key_code_scales = data<float>(scales);
            a.out = data<int32_t>(lists);
            a.counts = data<int32_t>(counts);
            a.Nq = q.fresh;
            a.H = q.heads;
            raise_on(aa_page_select(&a, c10::cuda::getCurrentCUDAStream(device.index()).stream()), "select_pages");
        }
        return pair(lists, counts);
    });
}

// (dict of status words by device index, function that makes one)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(args[0]) || !PyCallable_Check(args[1])) {
        PyErr_SetString(PyExc_TypeError, "setup(dict, callable)");
        return nullptr;
    }
    Py_XSETREF(g_status_words, Py_NewRef(args[0]));
    Py_XSETREF(g_new_status_word, Py_NewRef(args[1]));
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(select)), METH_FASTCALL, nullptr},
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(setup)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() { return PyModule_Create(&module); }
