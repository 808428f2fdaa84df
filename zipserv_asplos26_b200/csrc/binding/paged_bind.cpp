// Python binding of the paged-cache operators: argument checks, outputs and
// workspaces from torch's allocator, and the C ABI calls on the current stream.
//
// A decode step makes some of these calls per layer, and their kernels take 3 to
// 10 us at small batches, so the call itself counts: written with the CPython and
// torch C++ APIs it takes 4 to 7 us, where the same checks in Python with ctypes
// took 16 to 20 (35 for sparse_attention). paged.py documents the functions.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../rows_meet.h"
#include "zipserv_b200.h"

namespace {

struct Refusal {
    std::string what;
};
struct PyRaised {};   // a Python exception is set

[[noreturn]] void refuse(std::string what) { throw Refusal{std::move(what)}; }
inline void need(bool ok, const char* what) {
    if (!ok) refuse(what);
}

const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kInt: return "int32";
        case at::kLong: return "int64";
        case at::kFloat: return "float32";
        case at::kChar: return "int8";
        case at::kBool: return "bool";
        case at::kBFloat16: return "bfloat16";
        case at::kHalf: return "float16";
        default: return c10::toString(t);
    }
}

bool given(PyObject* o) { return o != Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyRaised{};
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyRaised{};
    return v != 0;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyRaised{};
    return v;
}

template <typename T = void>
T* ptr(const at::Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Contiguous tensor of n elements on device `index`.
template <typename T = void>
T* vec(PyObject* o, int64_t n, at::ScalarType type, const char* name, int index) {
    if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.scalar_type() == type && t.is_cuda() && t.get_device() == index && t.numel() == n && t.is_contiguous())
            return ptr<T>(t);
    }
    refuse(std::string(name) + " must be a contiguous " + type_name(type) + " tensor of " + std::to_string(n) +
           " elements on cuda:" + std::to_string(index));
}

unsigned* err_word(PyObject* o, int index) {
    return given(o) ? vec<unsigned>(o, 1, at::kInt, "err", index) : nullptr;
}

struct Table {
    int* data;
    int64_t stride;
    int width;
};

Table block_table(PyObject* o, int64_t rows, int index) {
    if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == index && t.dim() == 2 &&
            t.size(0) == rows && t.size(1) > 0 && t.size(1) <= INT32_MAX && (t.stride(1) == 1 || t.size(1) == 1) &&
            (t.stride(0) >= t.size(1) || rows <= 1))
            return {ptr<int>(t), rows > 1 ? t.stride(0) : t.size(1), static_cast<int>(t.size(1))};
    }
    refuse("block_table must be int32 [" + std::to_string(rows) + ", width] on cuda:" + std::to_string(index) +
           " with contiguous rows");
}

void check_page_size(int64_t page) {
    need(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be a power of two from 16 to 256");
}

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? ZS_BF16 : t == at::kHalf ? ZS_FP16 : -1; }

ZsPagePool page_pool(const at::Tensor& t, const char* name) {
    const int dtype = dtype_code(t.scalar_type());
    if (dtype < 0 || t.dim() != 4)
        refuse(std::string(name) + " must be a bf16 or fp16 tensor [num_blocks, page_size, heads, dim]");
    check_page_size(t.size(1));
    if (t.numel() == 0 || t.size(0) > INT32_MAX || t.size(2) > INT32_MAX || t.size(3) > INT32_MAX)
        refuse(std::string(name) + " must not be empty");
    if (t.stride(3) != 1 || ((t.stride(0) | t.stride(1) | t.stride(2)) % 8) || !aligned16(t))
        refuse(std::string(name) + ": rows must be contiguous and 16-byte aligned");
    return {ptr(t), t.stride(0), t.stride(1), t.stride(2), static_cast<int>(t.size(0)), static_cast<int>(t.size(1)),
            static_cast<int>(t.size(2)), static_cast<int>(t.size(3)), dtype};
}

struct Pools {
    ZsPagePool k, v;
    int index;
    at::ScalarType type;
};

Pools page_pools(PyObject* ko, PyObject* vo) {
    const at::Tensor &k = cuda_tensor(ko, "k_pages"), &v = cuda_tensor(vo, "v_pages");
    Pools p{page_pool(k, "k_pages"), page_pool(v, "v_pages"), static_cast<int>(k.get_device()), k.scalar_type()};
    need(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && v.get_device() == p.index,
         "k_pages and v_pages must agree in shape, type and device");
    return p;
}

// q as contiguous, aligned [B, Hq, dim]; a [B, 1, Hq, dim] query is one token per sequence.
at::Tensor query(const at::Tensor& q, int64_t hkv, int64_t dim, at::ScalarType type, int index) {
    const bool four = q.dim() == 4 && q.size(1) == 1;
    if (!q.is_cuda() || q.get_device() != index || q.scalar_type() != type || !(four || q.dim() == 3) ||
        q.size(-1) != dim || q.size(-2) <= 0 || q.size(-2) % hkv || q.size(0) * q.size(-2) > INT32_MAX)
        refuse(std::string("q must be a ") + type_name(type) + " tensor [B, Hq, " + std::to_string(dim) +
               "] or [B, 1, Hq, " + std::to_string(dim) + "] on cuda:" + std::to_string(index) +
               " with Hq a multiple of " + std::to_string(hkv));
    at::Tensor r = q.is_contiguous() ? q : q.contiguous();
    return aligned16(r) ? r : r.clone();
}

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, int index) {
    return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(index)),
                                  std::nullopt);
}

// n elements of `type` from byte `offset` of a byte tensor's storage, as a tensor of their own.
at::Tensor part_of(const at::Tensor& block, int64_t offset, int64_t n, at::ScalarType type) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(block.storage()), block.key_set(),
                                                     c10::scalarTypeToTypeMeta(type));
    impl->set_storage_offset(offset / static_cast<int64_t>(c10::elementSize(type)));
    impl->set_sizes_contiguous(at::IntArrayRef(&n, 1));
    return at::Tensor(std::move(impl));
}

void* current_stream(int index) {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
}

// Makes device `index` current where it is not.
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    explicit OnDevice(int index) {
        if (c10::cuda::current_device() != index) guard.set_index(static_cast<c10::DeviceIndex>(index));
    }
};

// Sets a Python exception of class `module`.`type`.
void raise_as(const char* module, const char* type, const char* what) {
    PyObject* m = PyImport_ImportModule(module);
    PyObject* t = m ? PyObject_GetAttrString(m, type) : nullptr;
    if (t) PyErr_SetString(t, what);
    Py_XDECREF(t);
    Py_XDECREF(m);
}

template <typename A>
void call(int (*f)(const A*), const A& args, const char* name) {
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f(&args);
    Py_END_ALLOW_THREADS
    if (!status) return;
    raise_as("zipserv_asplos26_b200._lib", "ZipServError",
             (std::string(name) + " failed with cudaError " + std::to_string(status)).c_str());
    throw PyRaised{};
}

// ------------------------------------------------------------------ plan
PyObject* plan_step(PyObject* const* a) {
    PyTypeObject* type = reinterpret_cast<PyTypeObject*>(a[9]);      // StepPlan
    if (!PyType_Check(a[9]) || !PyType_IsSubtype(type, &PyTuple_Type)) refuse("plan_step needs its tuple class");
    const at::Tensor& lens = cuda_tensor(a[1], "seq_lens");
    const int index = static_cast<int>(lens.get_device());
    const int64_t R = lens.numel(), page = integer(a[5]), room = integer(a[6]);
    need(R >= 1 && R <= 8192, "plan_step takes 1 to 8192 requests");
    const Table table = block_table(a[0], R, index);
    need(R * table.width <= INT32_MAX, "block_table is too large");
    check_page_size(page);
    need(room >= 0 && room <= (int64_t{1} << 30), "max_tokens must be from 0 to 2**30");
    const int64_t cap = tensor(a[3], "free_blocks").numel();
    need(cap > 0 && cap <= INT32_MAX, "free_blocks must not be empty");
    ZsPlanStep p{};
    p.block_table = table.data;
    p.table_stride = table.stride;
    p.seq_lens = vec<int>(a[1], R, at::kInt, "seq_lens", index);
    p.new_lens = vec<int>(a[2], R, at::kInt, "new_lens", index);
    p.free_blocks = vec<int>(a[3], cap, at::kInt, "free_blocks", index);
    p.free_count = vec<int>(a[4], 1, at::kInt, "free_count", index);
    p.err = err_word(a[8], index);
    p.R = static_cast<int>(R);
    p.width = table.width;
    p.capacity = static_cast<int>(cap);
    p.page_size = static_cast<int>(page);
    p.max_tokens = static_cast<int>(room);
    OnDevice on(index);
    p.stream = current_stream(index);
    if (given(a[7])) {
        if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 7) refuse("out must be a StepPlan");
        auto item = [&](int i) { return PyTuple_GET_ITEM(a[7], i); };
        p.out_lens = vec<int>(item(0), R, at::kInt, "out.seq_lens", index);
        p.out_count = vec<int>(item(1), 1, at::kInt, "out.free_count", index);
        p.out_cu = vec<int>(item(2), R + 1, at::kInt, "out.cu_tokens", index);
        p.slots = vec<int64_t>(item(3), room, at::kLong, "out.slots", index);
        p.token_seq = vec<int>(item(4), room, at::kInt, "out.token_seq", index);
        p.positions = vec<int>(item(5), room, at::kInt, "out.positions", index);
        p.refused = vec<uint8_t>(item(6), R, at::kBool, "out.refused", index);
        need(p.out_lens != p.seq_lens && p.out_lens != p.new_lens && p.out_count != p.free_count,
             "out.seq_lens and out.free_count must be other buffers than the inputs");
        call(zs_plan_step, p, "zs_plan_step");
        Py_INCREF(a[7]);
        return a[7];
    }
    // one allocation for the seven outputs, each on a 16-byte boundary
    const int64_t sizes[7] = {R, 1, R + 1, room, room, room, R};
    const at::ScalarType types[7] = {at::kInt, at::kInt, at::kInt, at::kLong, at::kInt, at::kInt, at::kBool};
    int64_t at_byte[7], bytes = 0;
    for (int i = 0; i < 7; ++i) {
        at_byte[i] = bytes;
        bytes += (sizes[i] * static_cast<int64_t>(c10::elementSize(types[i])) + 15) / 16 * 16;
    }
    const at::Tensor block = fresh({bytes}, at::kByte, index);
    at::Tensor out[7];
    for (int i = 0; i < 7; ++i) out[i] = part_of(block, at_byte[i], sizes[i], types[i]);
    p.out_lens = ptr<int>(out[0]);
    p.out_count = ptr<int>(out[1]);
    p.out_cu = ptr<int>(out[2]);
    p.slots = ptr<int64_t>(out[3]);
    p.token_seq = ptr<int>(out[4]);
    p.positions = ptr<int>(out[5]);
    p.refused = ptr<uint8_t>(out[6]);
    call(zs_plan_step, p, "zs_plan_step");
    PyObject* r = type->tp_alloc(type, 7);           // a named tuple without a call of its class
    if (!r) throw PyRaised{};
    for (int i = 0; i < 7; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
    return r;
}

// -------------------------------------------------------- rotary and write
// [n, heads, dim] with contiguous, 16-byte aligned rows (copied when they are not).
at::Tensor rows(PyObject* o, int64_t n, int64_t dim, at::ScalarType type, const char* name, int index) {
    const at::Tensor& t = tensor(o, name);
    if (!t.is_cuda() || t.get_device() != index || t.scalar_type() != type || t.dim() != 3 || t.size(0) != n ||
        t.size(2) != dim || t.size(1) <= 0 || t.size(1) > INT32_MAX)
        refuse(std::string(name) + " must be a " + type_name(type) + " tensor [" + std::to_string(n) + ", heads, " +
               std::to_string(dim) + "] on cuda:" + std::to_string(index));
    if (t.stride(2) == 1 && !((t.stride(0) | t.stride(1)) % 8) && aligned16(t)) return t;
    at::Tensor c = t.contiguous();
    return aligned16(c) ? c : c.clone();
}

// The arguments of a rotary write, a[0 .. 11] of rope_write, into pools on device `index`
// of hkv heads of dim channels: fills p but for its pools. `type` is q's, k's and v's.
struct Turned {
    at::Tensor q, k, v, out;           // keeps copies and the output alive
};

template <class P>
Turned rope_args(PyObject* const* a, P& p, int64_t hkv, int64_t dim, at::ScalarType type, int index) {
    const at::Tensor& q0 = tensor(a[0], "q");
    need(q0.dim() == 3 && q0.size(0) <= INT32_MAX, "q must be [N, Hq, D]");
    const int64_t N = q0.size(0);
    Turned t;
    t.q = rows(a[0], N, dim, type, "q", index);
    t.k = rows(a[1], N, dim, type, "k", index);
    t.v = rows(a[2], N, dim, type, "v", index);
    const at::Tensor &q = t.q, &k = t.k, &v = t.v;
    need(k.size(1) == hkv && v.size(1) == hkv, "k and v must have the cache's heads");
    const at::Tensor& cs = tensor(a[4], "cos_sin");
    need(cs.scalar_type() == at::kFloat && cs.dim() == 2 && cs.is_cuda() && cs.get_device() == index &&
             cs.is_contiguous() && cs.size(0) > 0 && cs.size(0) <= INT32_MAX && aligned16(cs),
         "cos_sin must be a contiguous, 16-byte aligned float32 [rows, rot] tensor on the cache's device");
    const int64_t rot = cs.size(1);
    need(dim % 16 == 0 && dim <= 512, "head dim must be a multiple of 16 up to 512");
    need(rot > 0 && rot <= dim && rot % 16 == 0, "rot must be a multiple of 16, at most the head dim");
    const at::Tensor& pos = tensor(a[3], "positions");
    const int64_t axes = pos.dim() == 2 ? pos.size(0) : 1;
    need(pos.scalar_type() == at::kInt && pos.is_cuda() && pos.get_device() == index &&
             (pos.dim() == 1 || pos.dim() == 2) && pos.size(-1) == N && (N <= 1 || pos.stride(-1) == 1) && axes >= 1 &&
             axes <= 4,
         "positions must be int32 [N] or [axes, N] with contiguous rows and 1 to 4 axes");
    const char* bad_sections = "sections must give each axis its share of the rot / 2 pairs";
    if (given(a[8])) {
        PyObject* seq = PySequence_Fast(a[8], bad_sections);
        if (!seq) throw PyRaised{};
        int64_t sum = 0, n = PySequence_Fast_GET_SIZE(seq);
        bool ok = n == axes;
        for (int64_t i = 0; ok && i < n; ++i) {
            const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
            ok = x >= 0 && x <= rot;        // an error's -1 among the refused
            sum += x;
            p.sections[i] = static_cast<int>(x);
        }
        Py_DECREF(seq);
        if (PyErr_Occurred()) throw PyRaised{};
        need(ok && sum == rot / 2, bad_sections);
    } else {
        need(axes == 1, bad_sections);
        p.sections[0] = static_cast<int>(rot / 2);
    }
    p.slots = vec<int64_t>(a[5], N, at::kLong, "slots", index);
    p.err = err_word(a[11], index);
    p.interleaved = truth(a[9]);
    at::Tensor& out = t.out;
    if (given(a[10])) {
        out = tensor(a[10], "q_out");
        need(out.sizes() == q.sizes() && out.scalar_type() == type && out.is_cuda() &&
                 out.get_device() == index && out.is_contiguous() && aligned16(out),
             "q_out must be contiguous, aligned and of q's shape and type");
        need(zs::q_out_is_apart(out.data_ptr(), N, q.size(1), k.size(1), dim, q.data_ptr(), q.stride(0), q.stride(1),
                                k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1)),
             "q_out must be a contiguous q itself, or apart from q, k and v");
    } else {
        out = fresh({N, q.size(1), dim}, type, index);
    }
    p.stream = current_stream(index);
    p.q = ptr<uint16_t>(q);
    p.k = ptr<uint16_t>(k);
    p.v = ptr<uint16_t>(v);
    p.q_tok = q.stride(0);
    p.q_head = q.stride(1);
    p.k_tok = k.stride(0);
    p.k_head = k.stride(1);
    p.v_tok = v.stride(0);
    p.v_head = v.stride(1);
    p.q_out = ptr<uint16_t>(out);
    p.positions = ptr<int>(pos);
    p.pos_axis = axes > 1 ? pos.stride(0) : 0;
    p.cos_sin = ptr<float>(cs);
    p.N = static_cast<int>(N);
    p.Hq = static_cast<int>(q.size(1));
    p.axes = static_cast<int>(axes);
    p.table_rows = static_cast<int>(cs.size(0));
    p.rot = static_cast<int>(rot);
    return t;
}

// q_out as given, or the fresh output.
PyObject* turned_q(PyObject* q_out, Turned& t) {
    if (given(q_out)) {
        Py_INCREF(q_out);
        return q_out;
    }
    return THPVariable_Wrap(std::move(t.out));
}

PyObject* rope_write(PyObject* const* a) {
    const Pools pools = page_pools(a[6], a[7]);
    OnDevice on(pools.index);
    ZsRopeWrite p{};
    Turned t = rope_args(a, p, pools.k.num_heads, pools.k.head_dim, pools.type, pools.index);
    p.k_pool = pools.k;
    p.v_pool = pools.v;
    call(zs_rope_write, p, "zs_rope_write");
    return turned_q(a[10], t);
}

// ------------------------------------------------------------- attention
// The attention proper: fills p, but for its pools and dtype, from q3 (checked) and the
// rest, and calls it. Returns out as [B, Hq, D].
struct Attended {
    const at::Tensor& q3;
    at::ScalarType type;
    int index;
    int64_t page_size;
    Table table;
    const int *lens, *pages, *counts;
    int64_t top;
    unsigned* err;
};

template <class P>
at::Tensor attend(P& p, const Attended& x, PyObject* scale_o, PyObject* out_o, PyObject* lse_o, PyObject* most_o,
                  size_t (*workspace)(const P*), int (*f)(const P*), const char* name) {
    const int index = x.index;
    const at::Tensor& q3 = x.q3;
    const int64_t dim = q3.size(-1), B = q3.size(0), hq = q3.size(-2);
    need(static_cast<int64_t>(x.table.width) * x.page_size <= INT32_MAX,
         "block_table covers more than 2**31 - 1 tokens");
    const double scale = given(scale_o) ? number(scale_o) : 1.0 / std::sqrt(static_cast<double>(dim));
    need(std::isfinite(static_cast<float>(scale)), "softmax_scale must be finite");
    at::Tensor out;
    if (given(out_o)) {
        out = tensor(out_o, "out");
        need(out.numel() == q3.numel() && out.scalar_type() == x.type && out.is_cuda() &&
                 out.get_device() == index && out.is_contiguous() && aligned16(out),
             "out must be contiguous, aligned and of q's shape and type");
    } else {
        out = fresh(q3.sizes(), x.type, index);
    }
    if (given(most_o)) {
        const int64_t most = integer(most_o);
        need(most >= 0, "max_seqlen must not be negative");
        p.max_seqlen = static_cast<int>(std::min<int64_t>(most, INT32_MAX));
    }
    p.lse = given(lse_o) ? vec<float>(lse_o, B * hq, at::kFloat, "lse", index) : nullptr;
    p.stream = current_stream(index);
    p.q = ptr<uint16_t>(q3);
    p.block_table = x.table.data;
    p.table_stride = x.table.stride;
    p.seq_lens = x.lens;
    p.pages = x.pages;
    p.counts = x.counts;
    p.out = ptr<uint16_t>(out);
    p.err = x.err;
    p.B = static_cast<int>(B);
    p.Hq = static_cast<int>(hq);
    p.width = x.table.width;
    p.top = static_cast<int>(x.top);
    p.softmax_scale = static_cast<float>(scale);
    at::Tensor ws;
    if ((p.ws_bytes = workspace(&p)) > 0) {
        ws = fresh({static_cast<int64_t>(p.ws_bytes)}, at::kByte, index);
        p.ws = ptr(ws);
    }
    call(f, p, name);
    return out;
}

at::Tensor attend16(const Pools& pools, const at::Tensor& q3, const Table& table, const int* lens, const int* pages,
                    const int* counts, int64_t top, PyObject* scale_o, PyObject* out_o, PyObject* lse_o,
                    PyObject* most_o, unsigned* err) {
    ZsPagedAttention p{};
    p.k_pool = pools.k;
    p.v_pool = pools.v;
    return attend(p, Attended{q3, pools.type, pools.index, pools.k.page_size, table, lens, pages, counts, top, err},
                  scale_o, out_o, lse_o, most_o, zs_paged_attention_workspace, zs_paged_attention, "zs_paged_attention");
}

// The page lists of a call: pages [B, Hkv, top] and counts, or neither.
struct Lists {
    const int *pages, *counts;
    int64_t top;
};

Lists page_lists(PyObject* pages_o, PyObject* counts_o, int64_t B, int64_t hkv, int64_t page_size, int index) {
    need(given(pages_o) == given(counts_o), "pages and counts go together");
    if (!given(pages_o)) return {nullptr, nullptr, 0};
    const at::Tensor& t = tensor(pages_o, "pages");
    need(t.dim() == 3 && t.size(2) > 0 && t.size(2) * page_size <= INT32_MAX, "pages must be int32 [B, Hkv, top]");
    return {vec<int>(pages_o, B * hkv * t.size(2), at::kInt, "pages", index),
            vec<int>(counts_o, B * hkv, at::kInt, "counts", index), t.size(2)};
}

void check_attention_dim(const Pools& pools) {
    need(pools.k.head_dim == 64 || pools.k.head_dim == 128, "head dim must be 64 or 128");
}

PyObject* paged_attention(PyObject* const* a) {
    const Pools pools = page_pools(a[1], a[2]);
    check_attention_dim(pools);
    const int index = pools.index;
    const int64_t hkv = pools.k.num_heads;
    OnDevice on(index);
    const at::Tensor q3 = query(tensor(a[0], "q"), hkv, pools.k.head_dim, pools.type, index);
    const int64_t B = q3.size(0);
    const Table table = block_table(a[3], B, index);
    const int* lens = vec<int>(a[4], B, at::kInt, "seq_lens", index);
    const Lists l = page_lists(a[6], a[7], B, hkv, pools.k.page_size, index);
    at::Tensor out = attend16(pools, q3, table, lens, l.pages, l.counts, l.top, a[5], a[8], a[9], a[10],
                              err_word(a[11], index));
    return THPVariable_Wrap(std::move(out));
}

// ---------------------------------------------------------------- sparse
struct Bounds {
    int8_t* codes;
    float* scales;
};

Bounds bounds_buffers(PyObject* codes_o, PyObject* scales_o, int64_t nb, int64_t hkv, int64_t dim, int index) {
    Bounds b{vec<int8_t>(codes_o, nb * hkv * 2 * dim, at::kChar, "page_codes", index),
             vec<float>(scales_o, nb * hkv, at::kFloat, "page_scales", index)};
    const at::Tensor& t = THPVariable_Unpack(codes_o);
    if (t.dim() != 4 || t.size(0) != nb || t.size(1) != hkv || t.size(2) != 2 || t.size(3) != dim || !aligned16(t))
        refuse("page_codes must be int8 [" + std::to_string(nb) + ", " + std::to_string(hkv) + ", 2, " +
               std::to_string(dim) + "], 16-byte aligned");
    return b;
}

PyObject* page_bounds(PyObject* const* a) {
    const at::Tensor& k = cuda_tensor(a[0], "k_pages");
    ZsPageBounds p{};
    p.k_pool = page_pool(k, "k_pages");
    const int index = static_cast<int>(k.get_device());
    const int dim = p.k_pool.head_dim;
    need(dim == 64 || dim == 128 || dim == 256, "head dim must be 64, 128 or 256");
    const int64_t B = tensor(a[3], "seq_lens").numel(), most = integer(a[6]);
    need(B <= INT32_MAX, "too many sequences");
    const Table table = block_table(a[1], B, index);
    p.lens_before = vec<int>(a[2], B, at::kInt, "lens_before", index);
    p.seq_lens = vec<int>(a[3], B, at::kInt, "seq_lens", index);
    const Bounds b = bounds_buffers(a[4], a[5], p.k_pool.num_blocks, p.k_pool.num_heads, dim, index);
    need(most >= 0 && most <= INT32_MAX, "max_new must be from 0 to 2**31 - 1");
    const int64_t total = given(a[7]) ? integer(a[7]) : 0;
    need(total >= 0 && total <= INT32_MAX, "max_total must be from 0 to 2**31 - 1");
    if (given(a[7]) && total == 0) Py_RETURN_NONE;
    p.max_total = static_cast<int>(total);
    p.err = err_word(a[8], index);
    OnDevice on(index);
    p.stream = current_stream(index);
    p.block_table = table.data;
    p.table_stride = table.stride;
    p.codes = b.codes;
    p.scales = b.scales;
    p.B = static_cast<int>(B);
    p.width = table.width;
    p.max_new = static_cast<int>(most);
    call(zs_page_bounds, p, "zs_page_bounds");
    Py_RETURN_NONE;
}

struct Choice {
    at::Tensor pages, counts;
};

Choice choose(const at::Tensor& q3, const Bounds& b, int64_t nb, int64_t hkv, const Table& table, const int* lens,
              int64_t page, int64_t top, int64_t sinks, int64_t local, unsigned* err, int index) {
    const int64_t B = q3.size(0), hq = q3.size(-2);
    need(hq / hkv <= 128, "at most 128 query heads may share a KV head");
    need(table.width <= 32768, "at most 32768 pages per sequence");
    check_page_size(page);
    need(sinks >= 0 && local >= 1 && sinks <= INT32_MAX && local <= INT32_MAX && top >= sinks + local &&
             top <= INT32_MAX,
         "top_pages must cover sink_pages (>= 0) and local_pages (>= 1)");
    Choice c{fresh({B, hkv, top}, at::kInt, index), fresh({B, hkv}, at::kInt, index)};
    ZsSelectPages p{};
    p.stream = current_stream(index);
    p.q = ptr<uint16_t>(q3);
    p.codes = b.codes;
    p.scales = b.scales;
    p.block_table = table.data;
    p.table_stride = table.stride;
    p.seq_lens = lens;
    p.pages = ptr<int>(c.pages);
    p.counts = ptr<int>(c.counts);
    p.err = err;
    p.dtype = dtype_code(q3.scalar_type());
    p.B = static_cast<int>(B);
    p.Hq = static_cast<int>(hq);
    p.Hkv = static_cast<int>(hkv);
    p.D = static_cast<int>(q3.size(-1));
    p.num_blocks = static_cast<int>(nb);
    p.width = table.width;
    p.page_size = static_cast<int>(page);
    p.top = static_cast<int>(top);
    p.sinks = static_cast<int>(sinks);
    p.local = static_cast<int>(local);
    call(zs_select_pages, p, "zs_select_pages");
    return c;
}

PyObject* select_pages(PyObject* const* a) {
    const at::Tensor& codes = cuda_tensor(a[1], "page_codes");
    const int index = static_cast<int>(codes.get_device());
    need(codes.dim() == 4 && codes.size(0) > 0 && codes.size(0) <= INT32_MAX && codes.size(1) > 0,
         "page_codes must be int8 [num_blocks, Hkv, 2, D]");
    const int64_t nb = codes.size(0), hkv = codes.size(1), dim = codes.size(3);
    need(dim == 64 || dim == 128 || dim == 256, "head dim must be 64, 128 or 256");
    const at::Tensor& q = tensor(a[0], "q");
    need(dtype_code(q.scalar_type()) >= 0, "q must be bf16 or fp16");
    OnDevice on(index);
    const at::Tensor q3 = query(q, hkv, dim, q.scalar_type(), index);
    const Bounds b = bounds_buffers(a[1], a[2], nb, hkv, dim, index);
    const Table table = block_table(a[3], q3.size(0), index);
    const int* lens = vec<int>(a[4], q3.size(0), at::kInt, "seq_lens", index);
    Choice c = choose(q3, b, nb, hkv, table, lens, integer(a[5]), integer(a[6]), integer(a[7]), integer(a[8]),
                      err_word(a[9], index), index);
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(c.pages)), THPVariable_Wrap(std::move(c.counts)));
}

PyObject* sparse_attention(PyObject* const* a) {
    const Pools pools = page_pools(a[1], a[2]);
    check_attention_dim(pools);
    const int index = pools.index;
    const int64_t hkv = pools.k.num_heads, dim = pools.k.head_dim, nb = pools.k.num_blocks;
    OnDevice on(index);
    const at::Tensor q3 = query(tensor(a[0], "q"), hkv, dim, pools.type, index);
    const Bounds b = bounds_buffers(a[3], a[4], nb, hkv, dim, index);
    const Table table = block_table(a[5], q3.size(0), index);
    const int* lens = vec<int>(a[6], q3.size(0), at::kInt, "seq_lens", index);
    unsigned* err = err_word(a[12], index);
    const int64_t top = integer(a[7]);
    need(top > 0 && top <= INT32_MAX / pools.k.page_size, "top_pages must be positive, and cover less than 2**31 tokens");
    Choice c = choose(q3, b, nb, hkv, table, lens, pools.k.page_size, top, integer(a[8]), integer(a[9]), err, index);
    at::Tensor out = attend16(pools, q3, table, lens, ptr<int>(c.pages), ptr<int>(c.counts), top, a[10], a[11], Py_None,
                              Py_None, err);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(c.pages)),
                         THPVariable_Wrap(std::move(c.counts)));
}

// ------------------------------------------------------------ 4-bit cache
// codes uint8 [num_blocks, page_size, heads, dim / 2] and params bf16 [num_blocks,
// page_size, heads, 2, dim / group] of one pool.
ZsInt4Pool int4_pool(PyObject* pages, const char* name, const char* codes, const char* params) {
    const at::Tensor &c = cuda_tensor(PyTuple_GET_ITEM(pages, 0), codes), &t = cuda_tensor(PyTuple_GET_ITEM(pages, 1), params);
    if (c.scalar_type() != at::kByte || c.dim() != 4 || t.scalar_type() != at::kBFloat16 || t.dim() != 5 ||
        t.get_device() != c.get_device())
        refuse(std::string(name) + " must be uint8 codes [num_blocks, page_size, heads, dim / 2] and bfloat16 params [num_blocks, "
                   "page_size, heads, 2, dim / group] on one CUDA device");
    check_page_size(c.size(1));
    const int64_t dim = c.size(3) * 2, groups = t.size(4);
    need(dim == 64 || dim == 128, "head dim must be 64 or 128");
    need(groups > 0 && (groups * 32 == dim || groups * 64 == dim), "params must have a scale and a centre for every 32 or 64 channels");
    if (c.numel() == 0 || c.size(0) > INT32_MAX || c.size(2) > INT32_MAX) refuse(std::string(name) + " must not be empty");
    if (t.size(0) != c.size(0) || t.size(1) != c.size(1) || t.size(2) != c.size(2) || t.size(3) != 2)
        refuse(std::string(name) + ": codes and params must agree in blocks, page size and heads");
    if (c.stride(3) != 1 || (c.stride(0) | c.stride(1) | c.stride(2)) % 16 || !aligned16(c) ||
        (t.stride(4) != 1 && groups > 1) || t.stride(3) != groups ||
        (t.stride(0) | t.stride(1) | t.stride(2)) % (2 * groups) ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % (4 * groups))
        refuse(std::string(name) + ": rows must be contiguous and aligned (codes to 16 bytes, params to a row's)");
    return {ptr<uint8_t>(c), ptr<uint16_t>(t), c.stride(0), c.stride(1), c.stride(2), t.stride(0), t.stride(1),
            t.stride(2), static_cast<int>(c.size(0)), static_cast<int>(c.size(1)), static_cast<int>(c.size(2)),
            static_cast<int>(dim), static_cast<int>(dim / groups), 0};
}

struct Int4Pools {
    ZsInt4Pool k, v;
    int index;
};

// k and v, each (codes, params).
Int4Pools int4_pools(PyObject* ko, PyObject* vo) {
    need(PyTuple_Check(ko) && PyTuple_GET_SIZE(ko) == 2 && PyTuple_Check(vo) && PyTuple_GET_SIZE(vo) == 2,
         "k_pages and v_pages must be Int4Pages");
    Int4Pools p{int4_pool(ko, "k_pages", "k_pages.codes", "k_pages.params"),
                int4_pool(vo, "v_pages", "v_pages.codes", "v_pages.params"),
                static_cast<int>(THPVariable_Unpack(PyTuple_GET_ITEM(ko, 0)).get_device())};
    need(p.k.num_blocks == p.v.num_blocks && p.k.page_size == p.v.page_size && p.k.num_heads == p.v.num_heads &&
             p.k.head_dim == p.v.head_dim && p.k.group == p.v.group &&
             THPVariable_Unpack(PyTuple_GET_ITEM(vo, 0)).get_device() == p.index,
         "k_pages and v_pages must agree in shape and device");
    return p;
}

at::ScalarType half_type(const at::Tensor& t, const char* name) {
    if (dtype_code(t.scalar_type()) < 0) refuse(std::string(name) + " must be bf16 or fp16");
    return t.scalar_type();
}

PyObject* rope_write_int4(PyObject* const* a) {
    const Int4Pools pools = int4_pools(a[6], a[7]);
    const at::ScalarType type = half_type(tensor(a[0], "q"), "q");
    OnDevice on(pools.index);
    ZsRopeWriteInt4 p{};
    Turned t = rope_args(a, p, pools.k.num_heads, pools.k.head_dim, type, pools.index);
    p.k_pool = pools.k;
    p.v_pool = pools.v;
    p.dtype = dtype_code(type);
    call(zs_rope_write_int4, p, "zs_rope_write_int4");
    return turned_q(a[10], t);
}

// k_pages, v_pages, slots, dtype as one of ZS_BF16 and ZS_FP16, out (None or a pair), err.
PyObject* read_int4(PyObject* const* a) {
    const Int4Pools pools = int4_pools(a[0], a[1]);
    const int index = pools.index;
    const int64_t dtype = integer(a[3]);
    need(dtype == ZS_BF16 || dtype == ZS_FP16, "dtype must be bfloat16 or float16");
    const at::ScalarType type = dtype == ZS_BF16 ? at::kBFloat16 : at::kHalf;
    const at::Tensor& slots = tensor(a[2], "slots");
    const int64_t N = slots.numel();
    need(slots.dim() == 1 && N <= INT32_MAX, "slots must be int64 [N]");
    ZsReadInt4 p{};
    p.slots = vec<int64_t>(a[2], N, at::kLong, "slots", index);
    p.err = err_word(a[5], index);
    OnDevice on(index);
    at::Tensor out[2];
    for (int i = 0; i < 2; ++i) {
        if (given(a[4])) {
            need(PyTuple_Check(a[4]) && PyTuple_GET_SIZE(a[4]) == 2, "out must be a pair of tensors");
            out[i] = tensor(PyTuple_GET_ITEM(a[4], i), "out");
            need(out[i].dim() == 3 && out[i].size(0) == N && out[i].size(1) == pools.k.num_heads &&
                     out[i].size(2) == pools.k.head_dim && out[i].scalar_type() == type && out[i].is_cuda() &&
                     out[i].get_device() == index && out[i].is_contiguous() && aligned16(out[i]),
                 "out must be two contiguous, aligned tensors [N, heads, dim] of dtype on the cache's device");
        } else {
            out[i] = fresh({N, pools.k.num_heads, pools.k.head_dim}, type, index);
        }
    }
    p.k_out = ptr<uint16_t>(out[0]);
    p.v_out = ptr<uint16_t>(out[1]);
    const int64_t len = out[0].numel();
    need(!zs::rows_meet(p.k_out, 1, 1, len, len, len, p.v_out, len), "out must be two tensors apart from one another");
    p.stream = current_stream(index);
    p.k_pool = pools.k;
    p.v_pool = pools.v;
    p.N = static_cast<int>(N);
    p.dtype = static_cast<int>(dtype);
    call(zs_read_int4, p, "zs_read_int4");
    if (given(a[4])) {
        Py_INCREF(a[4]);
        return a[4];
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])));
}

PyObject* paged_attention_int4(PyObject* const* a) {
    const Int4Pools pools = int4_pools(a[1], a[2]);
    const int index = pools.index;
    const int64_t hkv = pools.k.num_heads;
    const at::Tensor& q = tensor(a[0], "q");
    const at::ScalarType type = half_type(q, "q");
    OnDevice on(index);
    const at::Tensor q3 = query(q, hkv, pools.k.head_dim, type, index);
    const int64_t B = q3.size(0);
    const Table table = block_table(a[3], B, index);
    const int* lens = vec<int>(a[4], B, at::kInt, "seq_lens", index);
    const Lists l = page_lists(a[6], a[7], B, hkv, pools.k.page_size, index);
    need(!given(a[5]) || std::fabs(number(a[5])) < 0x1p57, "softmax_scale must be below 2**57 in magnitude");
    for (const ZsInt4Pool* x : {&pools.k, &pools.v})
        need(std::max({x->codes_block, x->codes_token, x->codes_head}) <= UINT32_MAX &&
                 std::max({x->params_block, x->params_token, x->params_head}) <= UINT32_MAX / 2,
             "attention takes pools with strides below 2**32 bytes");
    ZsPagedAttentionInt4 p{};
    p.k_pool = pools.k;
    p.v_pool = pools.v;
    p.dtype = dtype_code(type);
    at::Tensor out = attend(p, Attended{q3, type, index, pools.k.page_size, table, lens, l.pages, l.counts, l.top,
                                        err_word(a[11], index)},
                            a[5], a[8], a[9], a[10], zs_paged_attention_int4_workspace, zs_paged_attention_int4,
                            "zs_paged_attention_int4");
    return THPVariable_Wrap(std::move(out));
}

// -------------------------------------------------------------- sampling
// A setting for all rows (a number), or a row each (a tensor of B elements).
const float* setting(PyObject* o, int64_t B, const char* name, int index, double& one) {
    if (THPVariable_Check(o)) return vec<float>(o, B, at::kFloat, name, index);
    one = number(o);
    return nullptr;
}

// logits, u, temperature, top_k, top_p, min_p, out, err
PyObject* sample(PyObject* const* a) {
    const at::Tensor& x = cuda_tensor(a[0], "logits");
    const int index = static_cast<int>(x.get_device());
    const at::ScalarType type = x.scalar_type();
    need(x.dim() == 2 && (type == at::kFloat || dtype_code(type) >= 0), "logits must be a bf16, fp16 or float32 tensor [B, V]");
    const int64_t B = x.size(0), V = x.size(1);
    need(V > 0 && V <= (1 << 20) && B <= INT32_MAX / 8, "at most 2**20 tokens a row, and one at least");
    need(x.stride(1) == 1 || V == 1, "logits must have contiguous rows");
    ZsSample p{};
    p.logits = ptr(x);
    p.row_stride = B > 1 ? x.stride(0) : V;
    p.u = vec<float>(a[1], B, at::kFloat, "u", index);
    p.temperature = setting(a[2], B, "temperature", index, p.temperature1);
    if (!THPVariable_Check(a[3])) {
        const int64_t k = integer(a[3]);
        need(k >= 0, "top_k must not be negative");
        p.top_k1 = static_cast<int>(std::min<int64_t>(k, INT32_MAX));
    } else {
        p.top_k = vec<int>(a[3], B, at::kInt, "top_k", index);
    }
    p.top_p = setting(a[4], B, "top_p", index, p.top_p1);
    p.min_p = setting(a[5], B, "min_p", index, p.min_p1);
    need(p.temperature || (p.temperature1 >= 0 && std::isfinite(p.temperature1)), "temperature must be 0 or more");
    need(p.top_p || (p.top_p1 >= 0 && p.top_p1 <= 1), "top_p must be from 0 to 1");
    need(p.min_p || (p.min_p1 >= 0 && p.min_p1 <= 1), "min_p must be from 0 to 1");
    at::Tensor out;
    OnDevice on(index);
    if (given(a[6])) {
        p.out = vec<int64_t>(a[6], B, at::kLong, "out", index);
    } else {
        out = fresh({B}, at::kLong, index);
        p.out = ptr<int64_t>(out);
    }
    p.err = err_word(a[7], index);
    p.stream = current_stream(index);
    p.B = static_cast<int>(B);
    p.V = static_cast<int>(V);
    p.dtype = type == at::kFloat ? ZS_FP32 : dtype_code(type);
    call(zs_sample, p, "zs_sample");
    if (given(a[6])) {
        Py_INCREF(a[6]);
        return a[6];
    }
    return THPVariable_Wrap(std::move(out));
}

// No C++ exception leaves a C entry: refusals are ValueErrors, the rest RuntimeErrors.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    try {
        return F(args);
    } catch (const PyRaised&) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
    } catch (const Refusal& r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
    } catch (const c10::OutOfMemoryError& e) {
        raise_as("torch", "OutOfMemoryError", e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

#define ZS_ENTRY(name, n) \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ZS_ENTRY(plan_step, 10),    ZS_ENTRY(rope_write, 12),  ZS_ENTRY(paged_attention, 12),
                         ZS_ENTRY(page_bounds, 9),  ZS_ENTRY(select_pages, 10), ZS_ENTRY(sparse_attention, 13),
                         ZS_ENTRY(rope_write_int4, 12), ZS_ENTRY(read_int4, 6), ZS_ENTRY(paged_attention_int4, 12),
                         ZS_ENTRY(sample, 8),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_native(void) { return PyModule_Create(&module); }
