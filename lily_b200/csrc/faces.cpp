// Python faces in C++ of the operators of a cache held to a budget and of those on numbers held in four bits: checks of arguments, what is allocated, the launch.
//
// A small call of these is over on the device in 3 to 6 us, and a face in Python, some seventy looks at its tensors and thirty numbers
// through ctypes, takes 13 to 15 us of the host; here it is 5 to 6.  The kernels stay what they are, C entries over raw pointers in a library
// of their own, whose addresses `bind` is given; this module looks at tensors, so it is built against torch's headers.
//
// Every function raises what ops.py raises: KernelError for arguments that do not fit and for what the kernels' own checks refuse, torch's
// errors for an allocation that fails.  No C++ exception leaves it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <sstream>
#include <string>
#include <tuple>
#include <vector>

namespace {

using at::Tensor;

constexpr int F32 = 0, BF16 = 1;          // the kernels' codes of element types

struct Refusal { std::string why; };
struct Raised {};                          // a Python error is set

PyObject* kernel_error = nullptr;

struct Entries {
    const char* (*last_error)();
    int (*axes_rope_write)(const void*, int, int, size_t, int, const void*, const void*, int, float, const float*, const float*, int, const int*, const int*, int, int,
                           const int*, const int*, const int*, int, int, void*, int, void*, int, int, int, int, int, int, void*);
    size_t (*decode_weighed_floats)(int, int, int, int, int, int, int);
    int (*decode_weighed)(const void*, const void*, float*, void*, const int*, int, const int*, float*, int, int, int, int, int, int, int, float, int, int, void*);
    int (*select_keys)(const float*, const int*, int, const int*, int*, int, int, int, int, int, int, int, int, int, void*);
    int (*move_keys)(void*, float*, const int*, int, const int*, int, const int*, int, int, int, int, int, int, int, int, void*);
    int (*key_weights)(const void*, const void*, float*, const int*, int, float*, int, const int*, const int*, int, int, int, int, int, float, int, int, void*);
    size_t (*key_weights_floats)(int, const int*, const int*, int, int, int, int);
    int (*key_weights_tc)(const void*, int, const void*, int, float*, const int*, int, float*, int, const int*, const int*, int, int, int, int, int, float, int, int, void*);
    size_t (*key_weights_tc_floats)(int, const int*, const int*, int, int, int);
    int (*key_weights_tc_takes)(int, int, int, int, float);
    // numbers held in four bits
    int (*linear4)(const void*, int, const void*, const void*, const void*, const void*, int, void*, int, int, int, int, int, void*);
    int (*linear4_many)(const void*, const void*, const void*, const void*, const void*, int, void*, int, int, int, int, int, void*);
    int (*linear4_many_within)(const void*, const void*, const void*, const void*, const void*, int, void*, int, int, int, int, int, int, void*);
    int (*weights4)(const void*, const void*, const void*, void*, int, int, int, int, void*);
    int (*write4)(const void*, int, int, const void*, const void*, int, double, const float*, const float*, int, const int*, int, const int*, const int*, int, int, void*, int, void*, int, int,
                  int, int, int, void*);
    int (*values4)(const void*, int, const int*, int, int, void*, int, int, int, int, const int*, const int*, int*, int, int, const unsigned*, void*);
    size_t (*decode4_floats)(int, int, int, int, int, int, int);
    int (*decode4)(const void*, const void*, void*, const int*, int, const int*, float*, int, int, int, int, int, int, int, float, int, void*);
    int (*halves4)(const void*, int, int, const void*, int, const int*, int, int, int, int, int, const int*, const int*, int, unsigned*, size_t, const int*, int, int*, void*, float*, void*);
    int (*halves4_tiles)();
    int (*prefill_tc_half)(const void*, const void*, void*, const int*, int, const int*, const int*, const int*, const int*, int, int, int, int, int, float, int, int, const unsigned*, const unsigned*, const float*, void*);
    int (*prefill_mma_half)(const void*, const void*, void*, const int*, int, const int*, const int*, const int*, const int*, int, int, int, int, int, float, const unsigned*, const unsigned*, const float*, void*);
} entry;

// ---- words ----
void say(std::ostringstream&) {}
template <typename A, typename... R>
void say(std::ostringstream& s, const A& a, const R&... rest) { s << a; say(s, rest...); }
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    say(s, a...);
    throw Refusal{s.str()};
}
std::string words(const std::vector<int64_t>& shape) {
    std::ostringstream s;
    s << '(';
    for (size_t i = 0; i < shape.size(); ++i) s << (i ? ", " : "") << shape[i];
    s << (shape.size() == 1 ? ",)" : ")");
    return s.str();
}
std::string words(at::IntArrayRef shape) { return words(shape.vec()); }
std::string words(const Tensor& t) { return std::string("torch.") + (t.scalar_type() == at::kFloat ? "float32" : t.scalar_type() == at::kBFloat16 ? "bfloat16" : t.scalar_type() == at::kInt ? "int32" : c10::toString(t.scalar_type())) + " " + words(t.sizes()); }

// ---- arguments ----
const Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) refuse("kernels take tensors, got ", Py_TYPE(o)->tp_name);
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse("lily_b200 kernels run on a CUDA device only; got a tensor on ", t.device().str());
    if (!t.is_contiguous()) refuse("kernels take contiguous tensors (shape ", words(t.sizes()), ", strides ", words(t.strides()), ")");
    return t;
}
const Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
long long whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
// A number that the kernels take as a 32-bit one.
int number(PyObject* o) {
    const long long v = whole(o);
    if (v < INT32_MIN || v > INT32_MAX) refuse("kernels take 32-bit sizes, got ", v);
    return (int)v;
}
int narrow(int64_t v) {
    if (v > INT32_MAX) refuse("kernels take 32-bit sizes, got ", v);
    return (int)v;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return (float)v;
}
int code_of(const Tensor& t) {
    if (t.scalar_type() == at::kFloat) return F32;
    if (t.scalar_type() == at::kBFloat16) return BF16;
    refuse("kernels take float32 or bfloat16 tensors, got ", words(t));
}
bool is(const Tensor& t, at::ScalarType k) { return t.scalar_type() == k; }
const int* ints(const Tensor& t, const char* name) {
    if (!is(t, at::kInt)) refuse(name, " must be int32, got ", words(t));
    return t.const_data_ptr<int>();
}
bool shaped(const Tensor& t, std::initializer_list<int64_t> want) {
    const auto have = t.sizes();
    return have.size() == want.size() && std::equal(have.begin(), have.end(), want.begin());
}
void layer_fits(const Tensor& kv, int64_t nkv, int64_t page, int64_t d) {
    const auto s = kv.sizes();
    if (s.size() != 5 || s[1] != 2 || s[2] != nkv || s[3] != page || s[4] != d)
        refuse("cache layer shape ", words(s), " does not fit kv_heads=", nkv, " page=", page, " d=", d);
}
// The width of a block table of so many requests.
int table_width(const char* what, const Tensor& t, int64_t requests, const char* name = "block_table") {
    if (t.dim() != 2 || t.size(0) != requests || t.size(1) < 1 || !is(t, at::kInt)) refuse(what, ": ", name, " is int32 [", requests, ", pages], got ", words(t));
    return narrow(t.size(1));
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// The kernels' own answer.
void done(const char* name, int code) {
    if (code != 0) refuse(name, ": ", entry.last_error());
}
template <typename F, typename... A>
int call(F f, A... a) {
    if (f == nullptr) refuse("the kernels are not bound");
    int code;
    Py_BEGIN_ALLOW_THREADS
    code = f(a...);
    Py_END_ALLOW_THREADS
    return code;
}

template <typename F>
PyObject* guarded(Py_ssize_t count, Py_ssize_t want, F&& f) {
    HANDLE_TH_ERRORS
    try {
        if (count != want) refuse("a face takes ", want, " arguments, got ", count);
        return f();
    } catch (const Refusal& r) {
        PyErr_SetString(kernel_error ? kernel_error : PyExc_RuntimeError, r.why.c_str());
        return nullptr;
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---- the faces ----

// qkv, q_gain, k_gain, eps, cos, sin, positions, pair_axis, places, token_req, block_table, kv_layer, nq, nkv, d, rotary_dim, page_size, q_out, row
PyObject* axes_rope_write(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 19, [&]() -> PyObject* {
        const Tensor &qkv = tensor(p[0]), &cos = tensor(p[4]), &sin = tensor(p[5]), &positions = tensor(p[6]), &pair_axis = tensor(p[7]), &places = tensor(p[8]),
                     &req = tensor(p[9]), &table = tensor(p[10]), &kv = tensor(p[11]);
        const Tensor *q_gain = maybe(p[1]), *k_gain = maybe(p[2]), *given = maybe(p[17]);
        const float eps = real(p[3]);
        const int nq = number(p[12]), nkv = number(p[13]), d = number(p[14]), rd = number(p[15]), page = number(p[16]), row = p[18] == Py_None ? 0 : number(p[18]);
        const int64_t ld = row ? row : ((int64_t)nq + 2 * (int64_t)nkv) * d, half = rd / 2;
        if (qkv.dim() < 2) refuse("axes_rope_write qkv: expected [tokens, ", ld, "], got ", words(qkv.sizes()));
        const int64_t n = qkv.size(-2);
        int64_t splits = 1, stride = 0;
        if (qkv.dim() == 3) {
            if (!is(qkv, at::kFloat) || qkv.size(2) != ld) refuse("axes_rope_write qkv: partial sums must be float32 [splits, ", n, ", ", ld, "], got ", words(qkv));
            splits = qkv.size(0);
            stride = n * ld;
        } else if (qkv.dim() != 2 || qkv.size(1) != ld) refuse("axes_rope_write qkv: expected [", n, ", ", ld, "], got ", words(qkv.sizes()));
        const int code = code_of(kv), in = code_of(qkv);
        if (in != code && in != F32) refuse("axes_rope_write: cache dtype ", words(kv), " differs from activations ", words(qkv));
        layer_fits(kv, nkv, page, d);
        if (!is(cos, at::kFloat) || !is(sin, at::kFloat) || cos.dim() != 2 || cos.size(1) != half || sin.sizes() != cos.sizes())
            refuse("axes_rope_write: rotation tables are float32 [positions, rotary_dim / 2]");
        if (positions.dim() != 2 || positions.size(1) != n || pair_axis.numel() != half)
            refuse("axes_rope_write: positions are [axes, ", n, "] and there is an axis for each of the ", half, " pairs; got ", words(positions.sizes()), " and ", pair_axis.numel());
        if (places.numel() != n || req.numel() != n || table.dim() != 2 || table.size(1) < 1) refuse("axes_rope_write: ", n, " tokens have a place and a request each");
        int gain = F32;
        if (q_gain || k_gain) {
            if (!q_gain || !k_gain || q_gain->scalar_type() != k_gain->scalar_type() || q_gain->numel() != d || k_gain->numel() != d)
                refuse("axes_rope_write: q and k gains come together, with one dtype and head_dim numbers each");
            gain = code_of(*q_gain);
        }
        if (given && (given->scalar_type() != kv.scalar_type() || given->numel() != n * nq * d)) refuse("axes_rope_write: q_out is [tokens, nq * d] in the cache's dtype");
        const int *at = ints(positions, "positions"), *axis = ints(pair_axis, "pair_axis"), *to = ints(places, "places"), *of = ints(req, "token_req"), *bt = ints(table, "block_table");
        Tensor q = given ? *given : at::empty({n, (int64_t)nq * d}, kv.options());
        done("lily_axes_rope_write",
             call(entry.axes_rope_write, qkv.const_data_ptr(), in, narrow(splits), (size_t)stride, narrow(ld), q_gain ? q_gain->const_data_ptr() : nullptr,
                  k_gain ? k_gain->const_data_ptr() : nullptr, gain, eps, cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), narrow(cos.size(0)), at, axis,
                  narrow(positions.size(0)), narrow(n), to, of, bt, narrow(table.size(0)), narrow(table.size(1)), kv.data_ptr(), narrow(kv.size(0)), q.data_ptr(), code, nq, nkv, d, rd, page, stream()));
        return THPVariable_Wrap(std::move(q));
    });
}

// q, kv_layer, weights, block_table, seq_lens, max_seq_len, nq, nkv, d, page_size, scale, out, scratch, polls
PyObject* attention_decode_weighed(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 14, [&]() -> PyObject* {
        const char* what = "attention_decode_weighed";
        const Tensor &q = tensor(p[0]), &kv = tensor(p[1]), &weights = tensor(p[2]), &table = tensor(p[3]), &lens = tensor(p[4]);
        const Tensor *given = maybe(p[11]), *room = maybe(p[12]);
        const int longest = number(p[5]), nq = number(p[6]), nkv = number(p[7]), d = number(p[8]), page = number(p[9]), polls = number(p[13]);
        const float scale = real(p[10]);
        const int64_t requests = q.dim() ? q.size(0) : 0;
        if (q.scalar_type() != kv.scalar_type() || q.numel() != requests * nq * d)
            refuse(what, ": queries are [requests, ", (int64_t)nq * d, "] in the cache's dtype, got ", words(q));
        const int code = code_of(q);
        layer_fits(kv, nkv, page, d);
        if (!is(weights, at::kFloat) || !shaped(weights, {kv.size(0), nkv, page}))
            refuse(what, ": weights are float32 [", kv.size(0), ", ", nkv, ", ", page, "], got ", words(weights));
        const int width = table_width(what, table, requests);
        if (lens.numel() != requests || !is(lens, at::kInt) || longest < 0 || longest > (int64_t)width * page)
            refuse(what, ": ", requests, " int32 lengths of up to ", longest, " places; the block table holds ", (int64_t)width * page);
        if (given && (given->scalar_type() != q.scalar_type() || given->numel() != q.numel())) refuse(what, ": out has the shape and dtype of q");
        if (entry.decode_weighed_floats == nullptr) refuse("the kernels are not bound");
        const int64_t need = (int64_t)entry.decode_weighed_floats(narrow(requests), nq, nkv, d, longest, page, code);
        if (room && (!is(*room, at::kFloat) || room->numel() < need)) refuse(what, ": scratch of ", need, " float32 needed");
        Tensor out = given ? *given : at::empty_like(q), scratch = room ? *room : at::empty({need}, weights.options());
        done("lily_attention_decode_weighed", call(entry.decode_weighed, q.const_data_ptr(), kv.const_data_ptr(), weights.data_ptr<float>(), out.data_ptr(), table.const_data_ptr<int>(), width,
                                                   lens.const_data_ptr<int>(), scratch.data_ptr<float>(), (int)requests, longest, nq, nkv, d, page, narrow(kv.size(0)), scale, code, polls, stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// weights, block_table, lengths, max_length, keep, first, recent
PyObject* select_keys(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 7, [&]() -> PyObject* {
        const Tensor &weights = tensor(p[0]), &table = tensor(p[1]), &lengths = tensor(p[2]);
        const int longest = number(p[3]), keep = number(p[4]), first = number(p[5]), recent = number(p[6]);
        const auto s = weights.sizes();
        if (!is(weights, at::kFloat) || (s.size() != 3 && s.size() != 4)) refuse("select_keys: weights are float32 [layers, pages, kv_heads, page_size], got ", words(weights));
        const size_t o = s.size() - 3;
        const int64_t layers = o ? s[0] : 1, pages = s[o], nkv = s[o + 1], page = s[o + 2], requests = lengths.numel();
        const int width = table_width("select_keys", table, requests);
        if (keep < 1 || first < 0 || recent < 0 || (int64_t)first + recent > keep) refuse("select_keys: the first ", first, " and the last ", recent, " places do not fit into ", keep);
        if (!is(lengths, at::kInt) || longest < 0 || longest > width * page)
            refuse("select_keys: int32 lengths of up to ", longest, " places; the block table holds ", width * page);
        Tensor kept = at::empty({layers, requests, nkv, (int64_t)keep}, lengths.options());
        done("lily_select_keys", call(entry.select_keys, weights.const_data_ptr<float>(), table.const_data_ptr<int>(), width, lengths.const_data_ptr<int>(), kept.data_ptr<int>(), narrow(layers),
                                      narrow(pages), narrow(requests), narrow(nkv), narrow(page), longest, keep, first, recent, stream()));
        return THPVariable_Wrap(std::move(kept));
    });
}

// kv, weights, block_table, kept, to_table
PyObject* move_keys(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 5, [&]() -> PyObject* {
        const Tensor &kv = tensor(p[0]), &table = tensor(p[2]), &kept = tensor(p[3]);
        const Tensor *weights = maybe(p[1]), *to = maybe(p[4]);
        const auto s = kv.sizes();
        if ((s.size() != 5 && s.size() != 6) || s[s.size() - 4] != 2 || kept.dim() != 4 || !is(kept, at::kInt))
            refuse("move_keys: a cache [layers, pages, 2, kv_heads, page_size, d] and int32 places [layers, requests, kv_heads, keep], got ", words(s), ", ", words(kept));
        const size_t o = s.size() - 5;
        const int64_t layers = o ? s[0] : 1, pages = s[o], nkv = s[o + 2], page = s[o + 3], d = s[o + 4], requests = kept.size(1);
        if (kept.size(0) != layers || kept.size(2) != nkv) refuse("move_keys: places of ", kept.size(0), " layers and ", kept.size(2), " kv heads for a cache of ", layers, " and ", nkv);
        if (weights && (!is(*weights, at::kFloat) || !(o ? shaped(*weights, {layers, pages, nkv, page}) : shaped(*weights, {pages, nkv, page}))))
            refuse("move_keys: weights are float32 [", layers, ", ", pages, ", ", nkv, ", ", page, "], got ", words(*weights));
        const int item = code_of(kv) == F32 ? 4 : 2, width = table_width("move_keys", table, requests), to_width = to ? table_width("move_keys", *to, requests, "to_table") : width;
        const int *from = table.const_data_ptr<int>(), *into = to ? to->const_data_ptr<int>() : from;
        done("lily_move_keys", call(entry.move_keys, kv.data_ptr(), weights ? weights->data_ptr<float>() : nullptr, from, width, into, to_width, kept.const_data_ptr<int>(), narrow(layers),
                                    narrow(pages), narrow(requests), narrow(nkv), narrow(page), narrow(d * item), narrow(kept.size(3)), (int)(into == from), stream()));
        Py_RETURN_NONE;
    });
}

// The lengths of portions, host numbers.
std::vector<int> lengths(PyObject* o) {
    PyObject* fast = PySequence_Fast(o, "lengths of portions are a sequence of numbers");
    if (!fast) throw Raised{};
    std::vector<int> v;
    try {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
        v.reserve(n);
        for (Py_ssize_t i = 0; i < n; ++i) v.push_back(number(PySequence_Fast_GET_ITEM(fast, i)));
    } catch (...) {
        Py_DECREF(fast);
        throw;
    }
    Py_DECREF(fast);
    return v;
}
// What portions need: whether the tcgen05 kernels take them, and the scratch.
struct Plan { bool tensor_cores; int64_t floats, tokens, longest; };
Plan plan(const std::vector<int>& prefix, const std::vector<int>& fresh, int nq, int nkv, int d, int page, float scale, int code, int observe, int most_scores) {
    if (entry.key_weights_tc_takes == nullptr) refuse("the kernels are not bound");
    bool fits = nkv >= 1 && nq >= 1 && nq % nkv == 0 && prefix.size() == fresh.size();
    Plan p{};
    for (size_t r = 0; fits && r < fresh.size(); ++r) {
        fits = prefix[r] >= 0 && fresh[r] >= 0;
        p.tokens += fresh[r];
        p.longest = std::max(p.longest, (int64_t)prefix[r] + fresh[r]);
    }
    if (!fits) refuse("attention_key_weights: portions of ", words(std::vector<int64_t>(fresh.begin(), fresh.end())), " behind ", words(std::vector<int64_t>(prefix.begin(), prefix.end())), ", ", nq, " query heads over ", nkv, " kv heads");
    // (the kernels round places and tokens up to whole tiles in 32 bits)
    if (std::max(p.longest, p.tokens) > INT32_MAX - 1024) refuse("attention_key_weights: kernels take 32-bit sizes, got ", p.longest, " places and ", p.tokens, " tokens");
    p.tensor_cores = code == BF16 && entry.key_weights_tc_takes(nq, nkv, d, page, scale);
    const int requests = (int)fresh.size();
    p.floats = (int64_t)(p.tensor_cores ? entry.key_weights_tc_floats(requests, prefix.data(), fresh.data(), observe, nq, nkv)
                                        : entry.key_weights_floats(requests, prefix.data(), fresh.data(), observe, nq, nkv, most_scores));
    if (p.tokens > 0 && p.floats == 0) refuse("attention_key_weights: too many tiles for one call, ", p.tokens, " tokens of up to ", p.longest, " places");
    return p;
}
int observed(PyObject* o) {
    if (o == Py_None) return 0;
    const int n = number(o);
    if (n < 1) refuse("attention_key_weights: the last ", n, " tokens cannot be heard");
    return n;
}

// prefix lengths, new lengths, nq, nkv, d, page_size, scale, bfloat16 or not, observe, scores kept at a time
PyObject* key_weights_scratch_floats(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 10, [&]() -> PyObject* {
        return PyLong_FromLongLong(plan(lengths(p[0]), lengths(p[1]), number(p[2]), number(p[3]), number(p[4]), number(p[5]), real(p[6]), number(p[7]) ? BF16 : F32, observed(p[8]), number(p[9])).floats);
    });
}

// q, kv_layer, weights, block_table, cu_seqlens, prefix_lens, prefix lengths, new lengths, nq, nkv, d, page_size, scale, observe, scratch, scores kept at a time, polls of the row
// and of the column kernel
PyObject* attention_key_weights(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 18, [&]() -> PyObject* {
        const char* what = "attention_key_weights";
        const Tensor &q = tensor(p[0]), &kv = tensor(p[1]), &weights = tensor(p[2]), &table = tensor(p[3]), &cu = tensor(p[4]), &cached = tensor(p[5]);
        const Tensor* room = maybe(p[14]);
        const std::vector<int> prefix = lengths(p[6]), fresh = lengths(p[7]);
        const int nq = number(p[8]), nkv = number(p[9]), d = number(p[10]), page = number(p[11]), observe = observed(p[13]), most_scores = number(p[15]), row_polls = number(p[16]), column_polls = number(p[17]);
        const float scale = real(p[12]);
        const int64_t requests = (int64_t)fresh.size();
        if ((int64_t)prefix.size() != requests || cu.numel() != requests + 1 || cached.numel() != requests || !is(cu, at::kInt) || !is(cached, at::kInt))
            refuse(what, ": ", requests, " portions have a prefix each and ", requests + 1, " offsets, int32");
        const int code = code_of(q);
        const Plan plan_ = plan(prefix, fresh, nq, nkv, d, page, scale, code, observe, most_scores);
        if (q.scalar_type() != kv.scalar_type() || q.dim() != 2 || q.size(1) != (int64_t)nq * d || q.size(0) < plan_.tokens)
            refuse(what, ": queries are [tokens, ", (int64_t)nq * d, "] in the cache's dtype, got ", words(q), " for ", plan_.tokens, " tokens");
        layer_fits(kv, nkv, page, d);
        if (!is(weights, at::kFloat) || !shaped(weights, {kv.size(0), nkv, page}))
            refuse(what, ": weights are float32 [", kv.size(0), ", ", nkv, ", ", page, "], got ", words(weights));
        const int width = table_width(what, table, requests);
        if (plan_.longest > (int64_t)width * page) refuse(what, ": ", plan_.longest, " places; the block table holds ", (int64_t)width * page);
        if (plan_.tokens == 0) Py_RETURN_FALSE;
        if (room && (!is(*room, at::kFloat) || room->numel() < plan_.floats)) refuse(what, ": scratch of ", plan_.floats, " float32 needed");
        Tensor scratch = room ? *room : at::empty({plan_.floats}, weights.options());
        if (plan_.tensor_cores)
            done("lily_key_weights_tc", call(entry.key_weights_tc, q.const_data_ptr(), narrow(q.size(0)), kv.const_data_ptr(), narrow(kv.size(0)), weights.data_ptr<float>(), table.const_data_ptr<int>(),
                                             width, scratch.data_ptr<float>(), (int)requests, prefix.data(), fresh.data(), observe, nq, nkv, d, page, scale, row_polls, column_polls,
                                             stream()));
        else
            done("lily_key_weights", call(entry.key_weights, q.const_data_ptr(), kv.const_data_ptr(), weights.data_ptr<float>(), table.const_data_ptr<int>(), width, scratch.data_ptr<float>(),
                                          (int)requests, prefix.data(), fresh.data(), observe, nq, nkv, d, page, scale, code, most_scores, stream()));
        Py_RETURN_TRUE;
    });
}

// KernelError, then the addresses of the entries in their order
PyObject* bind(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 12, [&]() -> PyObject* {
        void* at[11];
        for (int i = 0; i < 11; ++i) at[i] = (void*)(uintptr_t)whole(p[i + 1]);
        entry.last_error = (decltype(entry.last_error))at[0];
        entry.axes_rope_write = (decltype(entry.axes_rope_write))at[1];
        entry.decode_weighed_floats = (decltype(entry.decode_weighed_floats))at[2];
        entry.decode_weighed = (decltype(entry.decode_weighed))at[3];
        entry.select_keys = (decltype(entry.select_keys))at[4];
        entry.move_keys = (decltype(entry.move_keys))at[5];
        entry.key_weights = (decltype(entry.key_weights))at[6];
        entry.key_weights_floats = (decltype(entry.key_weights_floats))at[7];
        entry.key_weights_tc = (decltype(entry.key_weights_tc))at[8];
        entry.key_weights_tc_floats = (decltype(entry.key_weights_tc_floats))at[9];
        entry.key_weights_tc_takes = (decltype(entry.key_weights_tc_takes))at[10];
        Py_INCREF(p[0]);
        Py_XDECREF(kernel_error);
        kernel_error = p[0];
        Py_RETURN_NONE;
    });
}

// ---- numbers held in four bits ----

// All of a call's tensors lie on the current device, where its kernels run.
void here(std::initializer_list<const Tensor*> all) {
    const int device = c10::cuda::current_device();
    for (const Tensor* t : all)
        if (t && t->get_device() != device) refuse("kernels run on the current device, ", device, "; got a tensor on ", t->device().str());
}
// A layer of a cache held in four bits: uint8 [pages, kv_heads, 2, page_size (d / 2 + d / 16)].
void layer4_fits(const char* what, const Tensor& kv, int64_t nkv, int64_t page, int64_t d) {
    if (d < 64 || d > 256 || d % 64) refuse(what, ": heads of 64, 128, 192 or 256 features, not ", d);
    if (!is(kv, at::kByte) || kv.dim() != 4 || !shaped(kv, {kv.size(0), nkv, 2, page * (d / 2 + d / 16)}) || kv.size(0) < 1)
        refuse(what, ": a cache layer is uint8 [pages, ", nkv, ", 2, ", page * (d / 2 + d / 16), "], got ", words(kv));
}
struct Matrix4 { const Tensor &codes, &scales; const Tensor* zeros; int n, k, group; };
// codes, scales, zeros, n, k, group from p[0] on
Matrix4 matrix4(const char* what, PyObject* const* p) {
    const Matrix4 w{tensor(p[0]), tensor(p[1]), maybe(p[2]), number(p[3]), number(p[4]), number(p[5])};
    if (w.n < 1 || w.k < 1 || w.n > INT32_MAX - 256 || w.k > INT32_MAX - 256 || (w.group != 32 && w.group != 64 && w.group != 128) || w.k % w.group)
        refuse(what, ": a matrix [", w.n, ", ", w.k, "] does not come in groups of ", w.group, " columns (32, 64 or 128)");
    const int64_t rows = (w.n + 127) / 128, tiles = (w.k + 127) / 128, groups = tiles * 128 / w.group;
    if (!is(w.codes, at::kByte) || !shaped(w.codes, {rows, tiles, 128, 64})) refuse(what, ": codes are uint8 [", rows, ", ", tiles, ", 128, 64], got ", words(w.codes));
    if (!is(w.scales, at::kBFloat16) || !shaped(w.scales, {rows, groups, 128})) refuse(what, ": scales are bfloat16 [", rows, ", ", groups, ", 128], got ", words(w.scales));
    if (w.zeros && (!is(*w.zeros, at::kByte) || w.zeros->sizes() != w.scales.sizes())) refuse(what, ": zero points are uint8 ", words(w.scales.sizes()), ", got ", words(*w.zeros));
    return w;
}

// x, codes, scales, zeros, n, k, group, bias, whether the result is float32 whatever x is, tokens from which on tcgen05 multiplies(, how often its waits ask)
PyObject* linear4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count == 11 ? 10 : count, 10, [&]() -> PyObject* {
        const Tensor& x = tensor(p[0]);
        const Matrix4 w = matrix4("linear4", p + 1);
        const Tensor* bias = maybe(p[7]);
        const int code = code_of(x), wide = code == F32 || PyObject_IsTrue(p[8]);
        if (x.dim() != 2 || x.size(1) != w.k) refuse("linear4: x ", words(x), " against a matrix [", w.n, ", ", w.k, "]");
        if (bias && (bias->dim() != 1 || bias->numel() != w.n || (code_of(*bias) == BF16 && code == F32))) refuse("linear4: a bias of ", w.n, " numbers, got ", words(*bias));
        here({&x, &w.codes, &w.scales, w.zeros, bias});
        Tensor out = at::empty({x.size(0), (int64_t)w.n}, x.options().dtype(wide ? at::kFloat : at::kBFloat16));
        if (code == BF16 && x.size(0) >= number(p[9])) {
            if (count == 11)
                done("lily_linear4_many", call(entry.linear4_many_within, x.const_data_ptr(), w.codes.const_data_ptr(), w.scales.const_data_ptr(), w.zeros ? w.zeros->const_data_ptr() : nullptr,
                                               bias ? bias->const_data_ptr() : nullptr, bias ? (int)(code_of(*bias) == F32) : 0, out.data_ptr(), wide, narrow(x.size(0)), w.n, w.k, w.group,
                                               number(p[10]), stream()));
            else done("lily_linear4_many", call(entry.linear4_many, x.const_data_ptr(), w.codes.const_data_ptr(), w.scales.const_data_ptr(), w.zeros ? w.zeros->const_data_ptr() : nullptr,
                                           bias ? bias->const_data_ptr() : nullptr, bias ? (int)(code_of(*bias) == F32) : 0, out.data_ptr(), wide, narrow(x.size(0)), w.n, w.k, w.group, stream()));
            return THPVariable_Wrap(std::move(out));
        }
        done("lily_linear4", call(entry.linear4, x.const_data_ptr(), code, w.codes.const_data_ptr(), w.scales.const_data_ptr(), w.zeros ? w.zeros->const_data_ptr() : nullptr,
                                  bias ? bias->const_data_ptr() : nullptr, bias ? (int)(code_of(*bias) == F32) : 0, out.data_ptr(), wide, narrow(x.size(0)), w.n, w.k, w.group, stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// codes, scales, zeros, n, k, group, whether float32
PyObject* weights4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 7, [&]() -> PyObject* {
        const Matrix4 w = matrix4("weights4", p);
        const bool wide = PyObject_IsTrue(p[6]);
        here({&w.codes, &w.scales, w.zeros});
        Tensor out = at::empty({(int64_t)w.n, (int64_t)w.k}, w.scales.options().dtype(wide ? at::kFloat : at::kBFloat16));
        done("lily_weights4", call(entry.weights4, w.codes.const_data_ptr(), w.scales.const_data_ptr(), w.zeros ? w.zeros->const_data_ptr() : nullptr, out.data_ptr(), wide ? F32 : BF16, w.n, w.k,
                                   w.group, stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// qkv, q_gain, k_gain, eps, cos, sin, positions, token_req, block_table, kv_layer, nq, nkv, d, rotary_dim, page_size, q_out
PyObject* qk_norm_rope_write4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 16, [&]() -> PyObject* {
        const char* what = "qk_norm_rope_write4";
        const Tensor &qkv = tensor(p[0]), &positions = tensor(p[6]), &req = tensor(p[7]), &table = tensor(p[8]), &kv = tensor(p[9]);
        const Tensor *q_gain = maybe(p[1]), *k_gain = maybe(p[2]), *cos = maybe(p[4]), *sin = maybe(p[5]), *given = maybe(p[15]);
        const double eps = PyFloat_AsDouble(p[3]);
        if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
        const int nq = number(p[10]), nkv = number(p[11]), d = number(p[12]), rd = number(p[13]), page = number(p[14]);
        if (nq < 1 || nkv < 1 || page < 1) refuse(what, ": ", nq, " query and ", nkv, " kv heads, pages of ", page, " places");
        layer4_fits(what, kv, nkv, page, d);
        const int64_t ld = ((int64_t)nq + 2 * (int64_t)nkv) * d;
        if (qkv.dim() != 2 || qkv.size(1) != ld) refuse(what, ": qkv is [tokens, ", ld, "], got ", words(qkv));
        const int64_t n = qkv.size(0);
        const int code = code_of(qkv);
        if (rd < 0 || rd > d || rd % 2 || (rd && (!cos || !sin))) refuse(what, ": rotary_dim ", rd, " does not fit head_dim ", d, ", or has no tables");
        if (rd && (!is(*cos, at::kFloat) || !is(*sin, at::kFloat) || cos->dim() != 2 || cos->size(0) < 1 || cos->size(1) != rd / 2 || sin->sizes() != cos->sizes()))
            refuse(what, ": rotation tables are float32 [positions, rotary_dim / 2]");
        if (positions.numel() != n || req.numel() != n || table.dim() != 2 || table.size(1) < 1) refuse(what, ": ", n, " tokens have a position and a request each, and there is a block table");
        int gain = F32;
        if (q_gain || k_gain) {
            if (!q_gain || !k_gain || q_gain->scalar_type() != k_gain->scalar_type() || q_gain->numel() != d || k_gain->numel() != d)
                refuse(what, ": q and k gains come together, with one dtype and head_dim numbers each");
            gain = code_of(*q_gain);
        }
        const bool rounded = given && code == F32 && is(*given, at::kBFloat16);
        if (given && ((given->scalar_type() != qkv.scalar_type() && !rounded) || given->numel() != n * nq * d)) refuse(what, ": q_out is [tokens, nq * d] in the dtype of qkv, or bfloat16");
        const int *at = ints(positions, "positions"), *of = ints(req, "token_req"), *bt = ints(table, "block_table");
        here({&qkv, q_gain, k_gain, cos, sin, &positions, &req, &table, &kv, given});
        Tensor q = given ? *given : at::empty({n, (int64_t)nq * d}, qkv.options());
        done("lily_qk_norm_rope_write4",
             call(entry.write4, qkv.const_data_ptr(), rounded ? 2 : code, narrow(ld), q_gain ? q_gain->const_data_ptr() : nullptr, k_gain ? k_gain->const_data_ptr() : nullptr, gain, eps,
                  rd ? cos->const_data_ptr<float>() : nullptr, rd ? sin->const_data_ptr<float>() : nullptr, rd ? narrow(cos->size(0)) : 0, at, narrow(n), of, bt, narrow(table.size(0)),
                  narrow(table.size(1)), kv.data_ptr(), narrow(kv.size(0)), q.data_ptr(), nq, nkv, d, rd, page, stream()));
        return THPVariable_Wrap(std::move(q));
    });
}

// kv_layer, block_table, nkv, d, page_size, whether float32
PyObject* cache4_values(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 6, [&]() -> PyObject* {
        const Tensor &kv = tensor(p[0]), &table = tensor(p[1]);
        const int nkv = number(p[2]), d = number(p[3]), page = number(p[4]);
        const bool wide = PyObject_IsTrue(p[5]);
        if (nkv < 1 || page < 1) refuse("cache4_values: ", nkv, " kv heads, pages of ", page, " places");
        layer4_fits("cache4_values", kv, nkv, page, d);
        if (table.dim() != 2 || !is(table, at::kInt)) refuse("cache4_values: block_table is int32 [requests, pages], got ", words(table));
        here({&kv, &table});
        Tensor out = at::empty({table.size(0), table.size(1), 2, (int64_t)nkv, (int64_t)page, (int64_t)d}, kv.options().dtype(wide ? at::kFloat : at::kBFloat16));
        done("lily_cache4_values", call(entry.values4, kv.const_data_ptr(), narrow(kv.size(0)), table.const_data_ptr<int>(), narrow(table.size(0)), narrow(table.size(1)), out.data_ptr(),
                                        wide ? F32 : BF16, nkv, d, page, (const int*)nullptr, (const int*)nullptr, (int*)nullptr, 0, 0, (const unsigned*)nullptr, stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// q, kv_layer, block_table, seq_lens, max_seq_len, nq, nkv, d, page_size, scale, out, scratch
PyObject* attention_decode4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 12, [&]() -> PyObject* {
        const char* what = "attention_decode4";
        const Tensor &q = tensor(p[0]), &kv = tensor(p[1]), &table = tensor(p[2]), &lens = tensor(p[3]);
        const Tensor *given = maybe(p[10]), *room = maybe(p[11]);
        const int longest = number(p[4]), nq = number(p[5]), nkv = number(p[6]), d = number(p[7]), page = number(p[8]);
        const float scale = real(p[9]);
        if (nkv < 1 || nq < 1 || nq % nkv || page < 1) refuse(what, ": ", nq, " query heads over ", nkv, " kv heads, pages of ", page, " places");
        layer4_fits(what, kv, nkv, page, d);
        const int64_t requests = q.dim() ? q.size(0) : 0;
        const int code = code_of(q);
        if (q.dim() != 2 || q.size(1) != (int64_t)nq * d) refuse(what, ": queries are [requests, ", (int64_t)nq * d, "], got ", words(q));
        const int width = table_width(what, table, requests);
        if (lens.numel() != requests || !is(lens, at::kInt) || longest < 0 || longest > (int64_t)width * page)
            refuse(what, ": ", requests, " int32 lengths of up to ", longest, " places; the block table holds ", (int64_t)width * page);
        if (given && (given->scalar_type() != q.scalar_type() || given->numel() != q.numel())) refuse(what, ": out has the shape and dtype of q");
        here({&q, &kv, &table, &lens, given, room});
        if (entry.decode4_floats == nullptr) refuse("the kernels are not bound");
        const int64_t need = (int64_t)entry.decode4_floats(narrow(requests), nq, nkv, d, longest, page, code);
        if (room && (!is(*room, at::kFloat) || room->numel() < need)) refuse(what, ": scratch of ", need, " float32 needed");
        Tensor out = given ? *given : at::empty_like(q), scratch;
        float* floats = nullptr;
        if (need) {
            scratch = room ? *room : at::empty({need}, q.options().dtype(at::kFloat));
            floats = scratch.data_ptr<float>();
        }
        done("lily_attention_decode4", call(entry.decode4, q.const_data_ptr(), kv.const_data_ptr(), out.data_ptr(), table.const_data_ptr<int>(), width, lens.const_data_ptr<int>(), floats,
                                            (int)requests, longest, nq, nkv, d, page, narrow(kv.size(0)), scale, code, stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// How portions are cut: the requests, then the offsets, of tiles of ``rows`` new tokens in the order of the keys that they see, and the pages that portions see.
struct Cut4 { std::vector<int> tiles; int64_t pages, width; Tensor both; };
Cut4 cut4(const char* what, const std::vector<int>& prefix, const std::vector<int>& fresh, int page, int rows) {
    if (prefix.size() != fresh.size() || page < 1 || rows < 1) refuse(what, ": ", fresh.size(), " portions behind ", prefix.size(), " lengths, pages of ", page, " places");
    std::vector<std::tuple<int64_t, int, int>> tiles;
    Cut4 c{{}, 0, 0, {}};
    for (size_t r = 0; r < fresh.size(); ++r) {
        if (fresh[r] < 0 || prefix[r] < 0) refuse(what, ": a portion of ", fresh[r], " tokens behind ", prefix[r]);
        if (fresh[r] == 0) continue;
        const int64_t pages = ((int64_t)prefix[r] + fresh[r] + page - 1) / page;
        c.pages += pages;
        c.width = std::max(c.width, pages);
        for (int64_t at = 0; at < fresh[r]; at += rows) tiles.emplace_back(prefix[r] + at, (int)r, (int)at);
    }
    std::sort(tiles.begin(), tiles.end());
    const size_t n = tiles.size();
    c.tiles.resize(2 * n);
    for (size_t i = 0; i < n; ++i) c.tiles[i] = std::get<1>(tiles[i]), c.tiles[n + i] = std::get<2>(tiles[i]);
    return c;
}
// ... on the device: both[0] the requests, both[1] the offsets.
void cut_to(const char* what, Cut4& c, int device) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) refuse(what, ": a captured call's plan is made ahead of the capture");
    Tensor host = at::empty({2, (int64_t)c.tiles.size() / 2}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    std::copy(c.tiles.begin(), c.tiles.end(), host.data_ptr<int>());
    c.both = host.to(at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)device), /*non_blocking=*/true);
}

// lengths of prefixes, of portions, page_size, rows of a tile, the device's index -> (requests, offsets, pages, width)
PyObject* plan4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 5, [&]() -> PyObject* {
        Cut4 c = cut4("plan_prefill4", lengths(p[0]), lengths(p[1]), number(p[2]), number(p[3]));
        cut_to("plan_prefill4", c, number(p[4]));
        return Py_BuildValue("(NNLL)", THPVariable_Wrap(c.both.select(0, 0)), THPVariable_Wrap(c.both.select(0, 1)), (long long)c.pages, (long long)c.width);
    });
}

// q, kv_layer, block_table, cu_seqlens, prefix_lens, lengths of prefixes, of portions, nq, nkv, d, page_size, scale, out, a plan's (rows, requests, offsets, pages, width) or None, rows of a tile, the
// kernel: 0 neither, 1 mma.sync, 2 tcgen05 -> out; for 0 (out, requests, offsets, pages, width), nothing launched
PyObject* attention_prefill4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 16, [&]() -> PyObject* {
        const char* what = "attention_prefill4";
        const Tensor &q = tensor(p[0]), &kv = tensor(p[1]), &table = tensor(p[2]), &cu = tensor(p[3]), &prefix = tensor(p[4]);
        const std::vector<int> cached = lengths(p[5]), fresh = lengths(p[6]);
        const int nq = number(p[7]), nkv = number(p[8]), d = number(p[9]), page = number(p[10]), rows = number(p[14]), kernel = number(p[15]);
        const float scale = real(p[11]);
        const Tensor* given = maybe(p[12]);
        const int64_t requests = (int64_t)fresh.size();
        if (nkv < 1 || nq < 1 || nq % nkv || page < 1 || (int64_t)cached.size() != requests)
            refuse(what, ": ", requests, " portions behind ", cached.size(), " lengths, ", nq, " query heads over ", nkv, " kv heads, pages of ", page, " places");
        layer4_fits(what, kv, nkv, page, d);
        code_of(q);
        int64_t tokens = 0;
        for (size_t r = 0; r < fresh.size(); ++r) {
            if (fresh[r] < 0 || cached[r] < 0) refuse(what, ": a portion of ", fresh[r], " tokens behind ", cached[r]);
            tokens += fresh[r];
        }
        if (q.dim() != 2 || q.size(1) != (int64_t)nq * d || q.size(0) < tokens) refuse(what, ": queries are [tokens, ", (int64_t)nq * d, "], got ", words(q), " for ", tokens, " tokens");
        if (cu.numel() != requests + 1 || prefix.numel() != requests) refuse(what, ": ", requests, " portions have a prefix each and ", requests + 1, " offsets");
        const int *offsets = ints(cu, "cu_seqlens"), *behind = ints(prefix, "prefix_lens");
        const int width = requests ? table_width(what, table, requests) : 0;
        if (given && (given->scalar_type() != q.scalar_type() || given->sizes() != q.sizes())) refuse(what, ": out has the shape and dtype of q");
        if (!(scale > 0.f) || scale > 3.4e38f) refuse(what, ": a scale of ", scale);
        here({&q, &kv, &table, &cu, &prefix, given});
        if (entry.halves4_tiles == nullptr) refuse("the kernels are not bound");
        Cut4 c{{}, 0, 0, {}};
        Tensor req, start;                               // a plan's tiles; those of a call without one go with its first launch where they are few
        int64_t tiles = 0;
        if (p[13] == Py_None) {
            c = cut4(what, cached, fresh, page, rows);
            tiles = (int64_t)c.tiles.size() / 2;
            if (kernel == 0 || tiles > entry.halves4_tiles()) {
                cut_to(what, c, q.get_device());
                req = c.both.select(0, 0), start = c.both.select(0, 1);
                c.tiles.clear();
            }
        } else {
            if (!PyTuple_Check(p[13]) || PyTuple_GET_SIZE(p[13]) != 5) refuse(what, ": a plan is what plan_prefill4 gives");
            req = tensor(PyTuple_GET_ITEM(p[13], 1)), start = tensor(PyTuple_GET_ITEM(p[13], 2)), c.pages = whole(PyTuple_GET_ITEM(p[13], 3)), c.width = whole(PyTuple_GET_ITEM(p[13], 4));
            int64_t pages = 0, most = 0;
            for (size_t r = 0; r < fresh.size(); ++r) {
                const int64_t own = fresh[r] ? ((int64_t)cached[r] + fresh[r] + page - 1) / page : 0;
                pages += own;
                most = std::max(most, own);
                tiles += ((int64_t)fresh[r] + rows - 1) / rows;
            }
            if (whole(PyTuple_GET_ITEM(p[13], 0)) != rows || c.pages != pages || c.width != most || req.numel() != tiles || start.numel() != tiles)
                refuse(what, ": the plan is not one of these portions (", tiles, " tiles of ", rows, " tokens, ", pages, " pages)");
            ints(req, "a plan's requests"), ints(start, "a plan's offsets");
            here({&req, &start});
        }
        if (c.width > width) refuse(what, ": ", c.width, " pages of a request; the block table holds ", width);
        Tensor out = given ? *given : at::empty_like(q);
        if (kernel == 0) return Py_BuildValue("(NNNLL)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(req)), THPVariable_Wrap(std::move(start)), (long long)c.pages, (long long)c.width);
        if (!is(q, at::kBFloat16)) refuse(what, ": these kernels take bfloat16");
        if (tokens == 0) return THPVariable_Wrap(std::move(out));
        // the keys' and the values' spans and the block table of the numbers, zeros; the numbers of the pages; queries in half precision and what undoes their powers of two
        const int64_t spans_n = 2 * requests * nkv, words_n = spans_n + requests * c.width;
        Tensor zeroed = at::empty({words_n + (int64_t)c.tiles.size()}, q.options().dtype(at::kInt)), values = at::empty({c.pages, 2, (int64_t)nkv, (int64_t)page, (int64_t)d}, q.options());
        Tensor heads = at::empty_like(q), units = at::empty({q.size(0), (int64_t)nq}, q.options().dtype(at::kFloat));
        unsigned* spans = (unsigned*)zeroed.data_ptr<int>();
        const unsigned* value_spans = spans + requests * nkv;
        int* numbers = zeroed.data_ptr<int>() + spans_n;
        const int* bt = table.const_data_ptr<int>();
        const int n = narrow(q.size(0)), pages = narrow(c.pages), wide = narrow(c.width), r = narrow(requests), tiles_n = narrow(tiles), held = narrow(kv.size(0));
        int* own = c.tiles.empty() ? nullptr : numbers + requests * c.width;
        const int *tile_req = own ? own : req.const_data_ptr<int>(), *tile_start = own ? own + tiles_n : start.const_data_ptr<int>();
        done("lily_halves4", call(entry.halves4, q.const_data_ptr(), n, nq, kv.const_data_ptr(), held, bt, r, width, nkv, d, page, offsets, behind, wide, spans, (size_t)words_n * 4, (const int*)c.tiles.data(), own ? tiles_n : 0, own, heads.data_ptr(),
                                  units.data_ptr<float>(), stream()));
        done("lily_cache4_values", call(entry.values4, kv.const_data_ptr(), held, bt, r, width, values.data_ptr(), BF16, nkv, d, page, offsets, behind, numbers, wide, pages, (const unsigned*)spans, stream()));
        if (kernel == 2)
            done("lily_attention_prefill_tc_half", call(entry.prefill_tc_half, heads.const_data_ptr(), values.const_data_ptr(), out.data_ptr(), (const int*)numbers, wide, offsets, behind, tile_req, tile_start,
                                                        tiles_n, nq, nkv, d, page, scale, n, pages, (const unsigned*)spans, value_spans, units.const_data_ptr<float>(), stream()));
        else
            done("lily_attention_prefill_mma_half", call(entry.prefill_mma_half, heads.const_data_ptr(), values.const_data_ptr(), out.data_ptr(), (const int*)numbers, wide, offsets, behind, tile_req,
                                                         tile_start, tiles_n, nq, nkv, d, page, scale, (const unsigned*)spans, value_spans, units.const_data_ptr<float>(), stream()));
        return THPVariable_Wrap(std::move(out));
    });
}

// the addresses of the entries for numbers held in four bits, in their order
PyObject* bind4(PyObject*, PyObject* const* p, Py_ssize_t count) {
    return guarded(count, 12, [&]() -> PyObject* {
        void* at[12];
        for (int i = 0; i < 12; ++i) at[i] = (void*)(uintptr_t)whole(p[i]);
        entry.linear4 = (decltype(entry.linear4))at[0];
        entry.weights4 = (decltype(entry.weights4))at[1];
        entry.write4 = (decltype(entry.write4))at[2];
        entry.values4 = (decltype(entry.values4))at[3];
        entry.decode4_floats = (decltype(entry.decode4_floats))at[4];
        entry.decode4 = (decltype(entry.decode4))at[5];
        entry.linear4_many = (decltype(entry.linear4_many))at[6];
        entry.halves4 = (decltype(entry.halves4))at[7];
        entry.prefill_tc_half = (decltype(entry.prefill_tc_half))at[8];
        entry.prefill_mma_half = (decltype(entry.prefill_mma_half))at[9];
        entry.halves4_tiles = (decltype(entry.halves4_tiles))at[10];
        entry.linear4_many_within = (decltype(entry.linear4_many_within))at[11];
        Py_RETURN_NONE;
    });
}

#define FACE(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FACE(axes_rope_write), FACE(attention_decode_weighed), FACE(select_keys), FACE(move_keys), FACE(key_weights_scratch_floats), FACE(attention_key_weights),
                         FACE(bind), FACE(linear4), FACE(weights4), FACE(qk_norm_rope_write4), FACE(cache4_values), FACE(attention_decode4), FACE(plan4), FACE(attention_prefill4), FACE(bind4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lily_faces", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lily_faces(void) { return PyModule_Create(&module); }
