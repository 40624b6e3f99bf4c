// The paged cache's calls for torch: tensors checked, results allocated, arguments packed, the C ABI called.
//
// A decode step makes these calls for every layer, and its kernels take 2 to 10 us.  Asked for one by one from Python, what a call has to know of its tensors took longer than
// that (13 to 15 us of the host for a call; here 5 to 6).  Nothing is computed here: torch carries memory and streams, the library's addresses are given by
// init(), so that this file knows the ABI's structures and no symbol of the library.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "../../include/kvcomp_b200.h"

namespace {

PyObject *error_class = nullptr;
decltype(&kvc_page_plan) page_plan = nullptr;
decltype(&kvc_page_release) page_release = nullptr;
decltype(&kvc_rotary_store) rotary_store = nullptr;
decltype(&kvc_paged_attn) paged_attn = nullptr;
decltype(&kvc_paged_attn_rows) paged_attn_rows = nullptr;
decltype(&kvc_last_error) last_error = nullptr;
decltype(&kvc_rotary_store_codes) rotary_store_codes = nullptr;
decltype(&kvc_page_slots) page_slots = nullptr;
decltype(&kvc_page_shift) page_shift = nullptr;
decltype(&kvc_paged_rows) paged_rows = nullptr;
decltype(&kvc_paged_attn_codes) paged_attn_codes = nullptr;
decltype(&kvc_prefix_plan_words) prefix_plan_words = nullptr;
decltype(&kvc_prefix_plan) prefix_plan = nullptr;
decltype(&kvc_paged_attn_shared) paged_attn_shared = nullptr;

[[noreturn]] void fail(const std::string &why) {
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, why.c_str());
    throw python_error();
}

std::string shape_of(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) fail(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

// the device of a call's first tensor; all others have to lie there
int device_of(const at::Tensor &t, const char *name) {
    if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (kvcomp_b200 has no CPU path)");
    return t.get_device();
}

void here(const at::Tensor &t, const char *name, int device, at::ScalarType type) {
    if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != type)
        fail(std::string(name) + " must be " + c10::toString(type) + " on cuda:" + std::to_string(device) + ", got " + c10::toString(t.scalar_type()) + " on " + t.device().str());
}

// a contiguous vector of n words
void *words(PyObject *o, int64_t n, const char *name, int device, at::ScalarType type = at::kInt) {
    const at::Tensor &t = tensor(o, name);
    here(t, name, device, type);
    if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        fail(std::string(name) + " must be a contiguous vector of " + std::to_string(n) + ", got " + shape_of(t.sizes()));
    return t.data_ptr();
}

// a tensor of a shape whose last dimension is contiguous
const at::Tensor &rows(PyObject *o, at::IntArrayRef shape, at::ScalarType type, const char *name, int device) {
    const at::Tensor &t = tensor(o, name);
    here(t, name, device, type);
    if (t.sizes() != shape) fail(std::string(name) + " must be " + shape_of(shape) + ", got " + shape_of(t.sizes()));
    if (t.stride(-1) != 1 && t.size(-1) > 1 && t.numel() > 0) fail(std::string(name) + " must have its last dimension contiguous, got strides " + shape_of(t.strides()));
    return t;
}

int32_t value_type(const at::Tensor &t, const char *name) {
    if (t.scalar_type() == at::kHalf) return KVC_TYPE_FP16;
    if (t.scalar_type() == at::kBFloat16) return KVC_TYPE_BF16;
    fail(std::string(name) + " must be fp16 or bf16, got " + c10::toString(t.scalar_type()));
}

int64_t number(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
bool given(PyObject *o) { return o != Py_None; }
void count(Py_ssize_t n, Py_ssize_t want) { if (n != want) fail("kvc_torch: wrong number of arguments"); }

struct Table { int32_t *at; int64_t stride, width; };
Table table_of(PyObject *o, int64_t B, int device) {
    const at::Tensor &t = tensor(o, "table");
    here(t, "table", device, at::kInt);
    if (t.dim() != 2 || t.size(0) != B || (t.stride(1) != 1 && t.size(1) > 1 && B > 0))
        fail("table must be int32 [" + std::to_string(B) + ", pages of a request], rows contiguous, got " + shape_of(t.sizes()));
    return {static_cast<int32_t *>(t.data_ptr()), B > 1 ? t.stride(0) : t.size(1), t.size(1)};
}
int32_t *status_of(PyObject *o, int device) { return given(o) ? static_cast<int32_t *>(words(o, 1, "status", device)) : nullptr; }

// the call on the device's current stream, other threads running meanwhile (a full queue makes a launch wait)
template <typename Call, typename Args, typename... More>
void launch(Call *call, const Args &args, int device, const char *name, More... more) {
    if (!call) fail("kvc_torch: init() has not been called");
    const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)));
    const kvc_stream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call(&args, more..., stream);
    Py_END_ALLOW_THREADS
    if (rc != KVC_OK) fail(std::string(name) + " failed (code " + std::to_string(rc) + "): " + last_error());
}

at::Tensor ints(int64_t n, const at::Tensor &like) { return at::empty({n}, like.options()); }
// a part of a buffer of words, as a tensor: a tenth of what a tensor of its own, or the buffer's narrow(), takes
at::Tensor part(const at::Tensor &buffer, int64_t first, int64_t n) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
    impl->set_storage_offset(first);
    impl->set_sizes_contiguous({n});
    return at::Tensor(std::move(impl));
}
int32_t *int_at(const at::Tensor &t) { return static_cast<int32_t *>(t.data_ptr()); }

// tensors of the caller's that a call has written: autograd refuses to go back through what it had kept of them
void written(std::initializer_list<PyObject *> given_tensors) {
    for (PyObject *o : given_tensors) {
        if (!given(o)) continue;
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
}

PyObject *tuple(std::initializer_list<at::Tensor> parts) {
    PyObject *r = PyTuple_New(static_cast<Py_ssize_t>(parts.size()));
    if (!r) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor &t : parts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    return r;
}

// The type of a pool's rows: the other tensors' type, or, where there are scales, codes'.  The scales of [pages, page_size, heads, channels] are [pages, heads, page_size].
kvc_scales scales_of(const at::Tensor &pool, PyObject *k, PyObject *v, at::ScalarType &type, int device) {
    kvc_scales s = {};
    const bool codes = pool.scalar_type() == at::kChar || pool.scalar_type() == at::kFloat8_e4m3fn;
    if (!given(k) && !given(v)) {
        if (codes) fail("pools of codes need kscales and vscales");
        return s;
    }
    if (!given(k) || !given(v)) fail("kscales and vscales must be given together");
    if (!codes) fail(std::string("with scales the pools must be int8 or float8_e4m3fn, got ") + c10::toString(pool.scalar_type()));
    type = pool.scalar_type();
    s.codes = type == at::kChar ? KVC_CODES_INT8 : KVC_CODES_E4M3;
    const int64_t shape[3] = {pool.size(0), pool.size(2), pool.size(1)};
    const at::Tensor &ks = rows(k, shape, at::kFloat, "kscales", device), &vs = rows(v, shape, at::kFloat, "vscales", device);
    s.k = static_cast<float *>(ks.data_ptr()); s.k_page = ks.stride(0); s.k_head = ks.stride(1);
    s.v = static_cast<float *>(vs.data_ptr()); s.v_page = vs.stride(0); s.v_head = vs.stride(1);
    return s;
}

// lengths, new, table, free, head, page_size, tokens, out (six tensors or None), status
PyObject *py_page_plan(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const at::Tensor &lengths = tensor(args[0], "lengths"), &free_list = tensor(args[3], "free");
    const int device = device_of(lengths, "lengths");
    kvc_page_plan_args a = {};
    a.B = lengths.dim() == 1 ? lengths.size(0) : -1;
    a.lengths = static_cast<int32_t *>(words(args[0], a.B, "lengths", device));
    a.new_tokens = static_cast<int32_t *>(words(args[1], a.B, "new", device));
    const Table table = table_of(args[2], a.B, device);
    a.table = table.at; a.table_stride = table.stride; a.table_width = table.width;
    a.n_pages = free_list.numel();
    a.free_pages = static_cast<int32_t *>(words(args[3], a.n_pages, "free", device));
    a.head = static_cast<int32_t *>(words(args[4], 1, "head", device));
    a.page_size = number(args[5]);
    a.tokens = number(args[6]);
    if (a.tokens < 0) fail("tokens must not be negative, got " + std::to_string(a.tokens));
    a.status = status_of(args[8], device);
    PyObject *result = nullptr;
    if (given(args[7])) {
        if (!PyTuple_Check(args[7]) || PyTuple_GET_SIZE(args[7]) != 6) fail("out must be a PagePlan");
        const int64_t sizes[6] = {a.B, 1, a.B + 1, a.B, a.tokens, a.tokens};
        static const char *const names[6] = {"out.lengths", "out.head", "out.starts", "out.taken", "out.slots", "out.positions"};
        int32_t **const to[6] = {&a.lengths_out, &a.head_out, &a.starts, &a.taken, &a.slots, &a.positions};
        for (int i = 0; i < 6; i++) *to[i] = static_cast<int32_t *>(words(PyTuple_GET_ITEM(args[7], i), sizes[i], names[i], device));
        launch(page_plan, a, device, "kvc_page_plan");
        for (int i = 0; i < 6; i++) written({PyTuple_GET_ITEM(args[7], i)});
        result = Py_NewRef(Py_None);
    } else {
        const int64_t room = (a.tokens + 3) / 4 * 4;        // (slots and positions are written 16 bytes at a time)
        const at::Tensor all = ints(2 * room + 3 * a.B + 2, lengths), slots = part(all, 0, a.tokens), positions = part(all, room, a.tokens), out_lengths = part(all, 2 * room, a.B),
                         head = part(all, 2 * room + a.B, 1), starts = part(all, 2 * room + a.B + 1, a.B + 1), taken = part(all, 2 * room + 2 * a.B + 2, a.B);
        a.lengths_out = int_at(out_lengths); a.head_out = int_at(head); a.starts = int_at(starts); a.taken = int_at(taken);
        a.slots = int_at(slots); a.positions = int_at(positions);
        launch(page_plan, a, device, "kvc_page_plan");
        result = tuple({out_lengths, head, starts, taken, slots, positions});
    }
    written({args[2]});
    return result;
    END_HANDLE_TH_ERRORS
}

// lengths, done, table, free, head, page_size, out lengths or None, out head or None, status
PyObject *py_page_release(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const at::Tensor &lengths = tensor(args[0], "lengths"), &free_list = tensor(args[3], "free");
    const int device = device_of(lengths, "lengths");
    kvc_page_release_args a = {};
    a.B = lengths.dim() == 1 ? lengths.size(0) : -1;
    a.lengths = static_cast<int32_t *>(words(args[0], a.B, "lengths", device));
    a.done = static_cast<uint8_t *>(words(args[1], a.B, "done", device, at::kBool));
    const Table table = table_of(args[2], a.B, device);
    a.table = table.at; a.table_stride = table.stride; a.table_width = table.width;
    a.n_pages = free_list.numel();
    a.free_pages = static_cast<int32_t *>(words(args[3], a.n_pages, "free", device));
    a.head = static_cast<int32_t *>(words(args[4], 1, "head", device));
    a.page_size = number(args[5]);
    a.status = status_of(args[8], device);
    const at::Tensor all = ints(2 * a.B + 2, lengths);      // scratch of B + 1 words, lengths, head
    a.first = int_at(all);
    if (given(args[6])) {
        a.lengths_out = static_cast<int32_t *>(words(args[6], a.B, "out lengths", device));
        a.head_out = static_cast<int32_t *>(words(args[7], 1, "out head", device));
        launch(page_release, a, device, "kvc_page_release");
        written({args[3], args[6], args[7]});
        return PyTuple_Pack(2, args[6], args[7]);
    }
    const at::Tensor out_lengths = part(all, a.B + 1, a.B), head = part(all, 2 * a.B + 1, 1);
    a.lengths_out = int_at(out_lengths); a.head_out = int_at(head);
    launch(page_release, a, device, "kvc_page_release");
    written({args[3]});
    return tuple({out_lengths, head});
    END_HANDLE_TH_ERRORS
}

// q or None, k or None, v, positions, slots, frequencies or None, kpages, vpages, layout, factor, inverse, out or None, status, kscales or None, vscales or None; q's name for messages is x without k
PyObject *py_rotary_store(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 15);
    const bool has_q = given(args[0]), has_k = given(args[1]);
    const char *const q_name = has_k ? "q" : "x", *const first_name = has_k ? "k" : "x";
    const at::Tensor &first = tensor(has_k ? args[1] : args[0], first_name);
    const int device = device_of(first, first_name);
    if (first.dim() != 3) fail(std::string(first_name) + " must be [N, heads, D], got " + shape_of(first.sizes()));
    const at::ScalarType type = first.scalar_type();
    kvc_rotary_args a = {};
    kvc_scales scales = {};
    a.type = value_type(first, first_name);
    a.N = first.size(0); a.D = first.size(2);
    if (has_k) {
        a.Hkv = first.size(1);
        const at::Tensor &k = rows(args[1], first.sizes(), type, "k", device), &v = rows(args[2], first.sizes(), type, "v", device);
        const at::Tensor &pool = tensor(args[6], "kpages");
        if (pool.dim() != 4 || pool.size(2) != a.Hkv || pool.size(3) != a.D)
            fail("the pools must be [pages, page_size, " + std::to_string(a.Hkv) + ", " + std::to_string(a.D) + "], got " + shape_of(pool.sizes()));
        at::ScalarType of_pool = type;
        scales = scales_of(pool, args[13], args[14], of_pool, device);
        const at::Tensor &kp = rows(args[6], pool.sizes(), of_pool, "kpages", device), &vp = rows(args[7], pool.sizes(), of_pool, "vpages", device);
        a.k = k.data_ptr(); a.k_token = k.stride(0); a.k_head = k.stride(1);
        a.v = v.data_ptr(); a.v_token = v.stride(0); a.v_head = v.stride(1);
        a.kpages = kp.data_ptr(); a.kp_page = kp.stride(0); a.kp_row = kp.stride(1); a.kp_head = kp.stride(2);
        a.vpages = vp.data_ptr(); a.vp_page = vp.stride(0); a.vp_row = vp.stride(1); a.vp_head = vp.stride(2);
        a.n_pages = pool.size(0); a.page_size = pool.size(1);
        a.slots = static_cast<int32_t *>(words(args[4], a.N, "slots", device));
    }
    if (!given(args[8])) fail("layout must be 'half' or 'interleaved'");
    a.layout = static_cast<int32_t>(number(args[8]));
    a.factor = static_cast<float>(real(args[9]));
    a.inverse = PyObject_IsTrue(args[10]);
    if (given(args[5])) {
        const at::Tensor &f = tensor(args[5], "frequencies");
        const int64_t pairs = f.numel();
        if (2 * pairs > a.D) fail("frequencies must be float64[rotated channels / 2], at most " + std::to_string(a.D / 2));
        a.frequencies = static_cast<double *>(words(args[5], pairs, "frequencies", device, at::kDouble));
        a.positions = static_cast<int32_t *>(words(args[3], a.N, "positions", device));
        a.rotary = 2 * pairs;
    }
    a.status = status_of(args[12], device);
    const auto call = [&] {
        if (scales.codes) launch(rotary_store_codes, a, device, "kvc_rotary_store_codes", static_cast<const kvc_scales *>(&scales));
        else launch(rotary_store, a, device, "kvc_rotary_store");
    };
    if (!has_q) {
        call();
        written({args[6], args[7], args[13], args[14]});
        Py_RETURN_NONE;
    }
    const at::Tensor &q0 = tensor(args[0], q_name);
    if (q0.dim() != 3 || q0.size(0) != a.N || q0.size(2) != a.D)
        fail(std::string(q_name) + " must be [" + std::to_string(a.N) + ", heads, " + std::to_string(a.D) + "], got " + shape_of(q0.sizes()));
    const at::Tensor &q = rows(args[0], q0.sizes(), type, q_name, device);
    a.Hq = q.size(1);
    a.q = q.data_ptr(); a.q_token = q.stride(0); a.q_head = q.stride(1);
    const bool own = !given(args[11]);
    const at::Tensor out = own ? at::empty(q.sizes(), q.options()) : rows(args[11], q.sizes(), type, "out", device);
    a.q_out = out.data_ptr(); a.out_token = out.stride(0); a.out_head = out.stride(1);
    call();
    written({args[6], args[7], args[11], args[13], args[14]});
    return own ? THPVariable_Wrap(out) : Py_NewRef(args[11]);
    END_HANDLE_TH_ERRORS
}

// table, lengths, page_size, tokens, status -> (slots, starts)
PyObject *py_page_slots(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const at::Tensor &lengths = tensor(args[1], "lengths");
    const int device = device_of(lengths, "lengths");
    kvc_page_slots_args a = {};
    a.B = lengths.dim() == 1 ? lengths.size(0) : -1;
    a.lengths = static_cast<int32_t *>(words(args[1], a.B, "lengths", device));
    const Table table = table_of(args[0], a.B, device);
    a.table = table.at; a.table_stride = table.stride; a.table_width = table.width;
    a.page_size = number(args[2]);
    a.tokens = number(args[3]);
    if (a.tokens < 0) fail("tokens must not be negative, got " + std::to_string(a.tokens));
    a.status = status_of(args[4], device);
    const at::Tensor slots = ints(a.tokens, lengths), starts = ints(a.B + 1, lengths);
    a.slots = int_at(slots); a.starts = int_at(starts);
    launch(page_slots, a, device, "kvc_page_slots");
    return tuple({slots, starts});
    END_HANDLE_TH_ERRORS
}

// starts, first, positions: positions of each request's rows go up by first, in place
PyObject *py_page_shift(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 3);
    const at::Tensor &first = tensor(args[1], "first"), &positions = tensor(args[2], "positions");
    const int device = device_of(positions, "positions");
    kvc_page_shift_args a = {};
    a.B = first.dim() == 1 ? first.size(0) : -1;
    a.tokens = positions.numel();
    a.positions = static_cast<int32_t *>(words(args[2], a.tokens, "positions", device));
    a.first = static_cast<int32_t *>(words(args[1], a.B, "first", device));
    a.starts = static_cast<int32_t *>(words(args[0], a.B + 1, "starts", device));
    launch(page_shift, a, device, "kvc_page_shift");
    written({args[2]});
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kpages, vpages, slots, kscales or None, vscales or None, bfloat16 or not or None, out (two tensors) or None, status -> (k, v)
PyObject *py_paged_rows(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 8);
    const at::Tensor &pool = tensor(args[0], "kpages"), &slots = tensor(args[2], "slots");
    const int device = device_of(pool, "kpages");
    if (pool.dim() != 4) fail("the pools must be [pages, page_size, Hkv, D], got " + shape_of(pool.sizes()));
    kvc_paged_rows_args a = {};
    at::ScalarType type = pool.scalar_type(), of_rows = type;
    a.scales = scales_of(pool, args[3], args[4], type, device);
    if (a.scales.codes) {
        if (!given(args[5])) fail("dtype must be fp16 or bf16: codes are of neither");
        of_rows = PyObject_IsTrue(args[5]) ? at::kBFloat16 : at::kHalf;
    } else {
        value_type(pool, "kpages");
        if (given(args[5]) && (PyObject_IsTrue(args[5]) ? at::kBFloat16 : at::kHalf) != type) fail(std::string("dtype must be the pools', ") + c10::toString(type));
    }
    const at::Tensor &kp = rows(args[0], pool.sizes(), type, "kpages", device), &vp = rows(args[1], pool.sizes(), type, "vpages", device);
    a.type = of_rows == at::kHalf ? KVC_TYPE_FP16 : KVC_TYPE_BF16;
    a.N = slots.numel(); a.n_pages = pool.size(0); a.page_size = pool.size(1); a.Hkv = pool.size(2); a.D = pool.size(3);
    a.slots = static_cast<int32_t *>(words(args[2], a.N, "slots", device));
    a.kpages = kp.data_ptr(); a.kp_page = kp.stride(0); a.kp_row = kp.stride(1); a.kp_head = kp.stride(2);
    a.vpages = vp.data_ptr(); a.vp_page = vp.stride(0); a.vp_row = vp.stride(1); a.vp_head = vp.stride(2);
    a.status = status_of(args[7], device);
    const int64_t shape[3] = {a.N, a.Hkv, a.D};
    const bool own = !given(args[6]);
    if (!own && (!PyTuple_Check(args[6]) || PyTuple_GET_SIZE(args[6]) != 2)) fail("out must be a tuple of two tensors");
    const at::Tensor k = own ? at::empty(shape, pool.options().dtype(of_rows)) : rows(PyTuple_GET_ITEM(args[6], 0), shape, of_rows, "out[0]", device);
    const at::Tensor v = own ? at::empty(shape, pool.options().dtype(of_rows)) : rows(PyTuple_GET_ITEM(args[6], 1), shape, of_rows, "out[1]", device);
    a.k_out = k.data_ptr(); a.k_token = k.stride(0); a.k_head = k.stride(1);
    a.v_out = v.data_ptr(); a.v_token = v.stride(0); a.v_head = v.stride(1);
    launch(paged_rows, a, device, "kvc_paged_rows");
    if (own) return tuple({k, v});
    written({PyTuple_GET_ITEM(args[6], 0), PyTuple_GET_ITEM(args[6], 1)});
    return Py_NewRef(args[6]);
    END_HANDLE_TH_ERRORS
}

// q, kpages, vpages, table, lengths, scaling, window, out or None, return_lse, workspace, status, starts or None, kscales or None, vscales or None, a prefix plan or None
PyObject *py_paged_attn(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 15);
    const at::Tensor &q0 = tensor(args[0], "q"), &pool = tensor(args[1], "kpages");
    const int device = device_of(q0, "q");
    kvc_paged_attn_args a = {};
    a.type = value_type(q0, "q");
    const at::ScalarType type = q0.scalar_type();
    if (q0.dim() != 3 || pool.dim() != 4 || pool.size(3) != q0.size(2))
        fail("q must be [B, Hq, D], the pools [pages, page_size, Hkv, D], got " + shape_of(q0.sizes()) + " and " + shape_of(pool.sizes()));
    at::ScalarType of_pool = type;
    const kvc_scales scales = scales_of(pool, args[12], args[13], of_pool, device);
    const at::Tensor &q = rows(args[0], q0.sizes(), type, "q", device), &kp = rows(args[1], pool.sizes(), of_pool, "kpages", device), &vp = rows(args[2], pool.sizes(), of_pool, "vpages", device);
    const bool by_row = given(args[11]), with_prefix = given(args[14]);
    if (with_prefix && scales.codes) fail("prefixes of pools of codes are not attended");
    const at::Tensor &lengths = tensor(args[4], "lengths");
    a.B = !by_row ? q.size(0) : lengths.dim() == 1 ? lengths.size(0) : -1;
    a.Hq = q.size(1); a.D = q.size(2);
    a.n_pages = pool.size(0); a.page_size = pool.size(1); a.Hkv = pool.size(2);
    a.q = q.data_ptr(); a.q_token = q.stride(0); a.q_head = q.stride(1);
    a.kpages = kp.data_ptr(); a.kp_page = kp.stride(0); a.kp_row = kp.stride(1); a.kp_head = kp.stride(2);
    a.vpages = vp.data_ptr(); a.vp_page = vp.stride(0); a.vp_row = vp.stride(1); a.vp_head = vp.stride(2);
    const Table table = table_of(args[3], a.B, device);
    a.table = table.at; a.table_stride = table.stride; a.table_width = table.width;
    a.lengths = static_cast<int32_t *>(words(args[4], a.B, "lengths", device));
    a.scaling = static_cast<float>(real(args[5]));
    a.window = number(args[6]);
    const at::Tensor &workspace = tensor(args[9], "workspace");
    a.workspace_bytes = workspace.numel();
    a.workspace = words(args[9], a.workspace_bytes, "workspace", device, at::kByte);
    a.status = status_of(args[10], device);
    const bool own = !given(args[7]);
    const at::Tensor out = own ? at::empty(q.sizes(), q.options()) : rows(args[7], q.sizes(), type, "out", device);
    a.out = out.data_ptr(); a.out_token = out.stride(0); a.out_head = out.stride(1);
    at::Tensor lse;
    if (PyObject_IsTrue(args[8])) {
        lse = at::empty({q.size(0), a.Hq}, q.options().dtype(at::kFloat));
        a.lse = static_cast<float *>(lse.data_ptr());
    }
    if (with_prefix)
        launch(paged_attn_shared, a, device, "kvc_paged_attn_shared", static_cast<const int32_t *>(words(args[14], prefix_plan_words ? prefix_plan_words(a.B) : 0, "plan", device)),
               by_row ? static_cast<const int32_t *>(words(args[11], a.B + 1, "starts", device)) : nullptr, q.size(0));
    else if (scales.codes)
        launch(paged_attn_codes, a, device, "kvc_paged_attn_codes", &scales, by_row ? static_cast<const int32_t *>(words(args[11], a.B + 1, "starts", device)) : nullptr, q.size(0));
    else if (by_row) launch(paged_attn_rows, a, device, "kvc_paged_attn_rows", static_cast<const int32_t *>(words(args[11], a.B + 1, "starts", device)), q.size(0));
    else launch(paged_attn, a, device, "kvc_paged_attn");
    written({args[7]});
    PyObject *const result = own ? THPVariable_Wrap(out) : Py_NewRef(args[7]);
    if (!lse.defined() || !result) return result;
    PyObject *const more = THPVariable_Wrap(lse);
    PyObject *const both = more ? PyTuple_Pack(2, result, more) : nullptr;
    Py_DECREF(result);
    Py_XDECREF(more);
    return both;
    END_HANDLE_TH_ERRORS
}

// parents, shared, out or None, status -> the plan
PyObject *py_prefix_plan(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 4);
    const at::Tensor &parents = tensor(args[0], "parents");
    const int device = device_of(parents, "parents");
    kvc_prefix_plan_args a = {};
    a.B = parents.dim() == 1 ? parents.size(0) : -1;
    a.parents = static_cast<int32_t *>(words(args[0], a.B, "parents", device));
    a.shared = static_cast<int32_t *>(words(args[1], a.B, "shared", device));
    if (!prefix_plan_words) fail("kvc_torch: init() has not been called");
    const int64_t all = prefix_plan_words(a.B);
    const bool own = !given(args[2]);
    const at::Tensor plan = own ? ints(all, parents) : (words(args[2], all, "out", device), tensor(args[2], "out"));
    a.plan = int_at(plan);
    a.status = status_of(args[3], device);
    launch(prefix_plan, a, device, "kvc_prefix_plan");
    if (own) return THPVariable_Wrap(plan);
    written({args[2]});
    return Py_NewRef(args[2]);
    END_HANDLE_TH_ERRORS
}

// device -> (handle of its current stream, number of the capture that it is in or 0)
PyObject *py_stream_of(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 1);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(number(args[0]))).stream();
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0;
    // (the legacy stream does not answer while another thread captures: it is in none then)
    if (cudaStreamGetCaptureInfo(stream, &status, &capture) != cudaSuccess) (void)cudaGetLastError(), status = cudaStreamCaptureStatusNone;
    return Py_BuildValue("KK", static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream)), status == cudaStreamCaptureStatusNone ? 0ull : capture);
    END_HANDLE_TH_ERRORS
}

// the error's class and the addresses of the library's entries
PyObject *py_init(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 15);
    error_class = Py_NewRef(args[0]);
    auto address = [&](int i) { return reinterpret_cast<void *>(static_cast<uintptr_t>(number(args[i]))); };
    page_plan = reinterpret_cast<decltype(page_plan)>(address(1));
    page_release = reinterpret_cast<decltype(page_release)>(address(2));
    rotary_store = reinterpret_cast<decltype(rotary_store)>(address(3));
    paged_attn = reinterpret_cast<decltype(paged_attn)>(address(4));
    paged_attn_rows = reinterpret_cast<decltype(paged_attn_rows)>(address(5));
    last_error = reinterpret_cast<decltype(last_error)>(address(6));
    rotary_store_codes = reinterpret_cast<decltype(rotary_store_codes)>(address(7));
    page_slots = reinterpret_cast<decltype(page_slots)>(address(8));
    page_shift = reinterpret_cast<decltype(page_shift)>(address(9));
    paged_rows = reinterpret_cast<decltype(paged_rows)>(address(10));
    paged_attn_codes = reinterpret_cast<decltype(paged_attn_codes)>(address(11));
    prefix_plan_words = reinterpret_cast<decltype(prefix_plan_words)>(address(12));
    prefix_plan = reinterpret_cast<decltype(prefix_plan)>(address(13));
    paged_attn_shared = reinterpret_cast<decltype(paged_attn_shared)>(address(14));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)> PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef methods[] = {{"init", fast<py_init>(), METH_FASTCALL, nullptr},
                         {"page_plan", fast<py_page_plan>(), METH_FASTCALL, nullptr},
                         {"page_release", fast<py_page_release>(), METH_FASTCALL, nullptr},
                         {"rotary_store", fast<py_rotary_store>(), METH_FASTCALL, nullptr},
                         {"paged_attn", fast<py_paged_attn>(), METH_FASTCALL, nullptr},
                         {"page_slots", fast<py_page_slots>(), METH_FASTCALL, nullptr},
                         {"page_shift", fast<py_page_shift>(), METH_FASTCALL, nullptr},
                         {"paged_rows", fast<py_paged_rows>(), METH_FASTCALL, nullptr},
                         {"prefix_plan", fast<py_prefix_plan>(), METH_FASTCALL, nullptr},
                         {"stream_of", fast<py_stream_of>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kvc_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kvc_torch() { return PyModule_Create(&module); }
