// kvsnap_amd.attention's calls: their arguments checked, their outputs allocated and the C entry points
// (include/kvsnap_attention.h) launched on the current stream of the cache's device.
//
// In C++ because a step makes these calls once a layer: checking eight tensors' shapes, types and devices from Python
// took 12 to 16 us of host time a call, more than the kernels of a decode step of few sequences run.  The entry
// points are those of the library that kvsnap_amd.native loads; `bind` is given their addresses.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kvsnap_attention.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <sstream>
#include <stdexcept>
#include <string>

namespace {

struct Library {
    decltype(&kvsnap_rotate) rotate;
    decltype(&kvsnap_append) append;
    decltype(&kvsnap_attend) attend;
    decltype(&kvsnap_attend_workspace_bytes) workspace_bytes;
    const char* (*error)();
} library;

struct Refused : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
struct Raised {};  // a Python error is set

template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
    std::ostringstream text;
    (text << ... << parts);
    throw Refused(text.str());
}

// ----------------------------------------------------------------- arguments

bool given(PyObject* object) { return object != Py_None; }

const at::Tensor& tensor(PyObject* object, const char* what) {
    if (!THPVariable_Check(object)) refuse(what, " must be a tensor");
    return THPVariable_Unpack(object);
}

int64_t whole(PyObject* object) {
    const int64_t value = PyLong_AsLongLong(object);
    if (value == -1 && PyErr_Occurred()) throw Raised{};
    return value;
}

bool truth(PyObject* object) {
    const int value = PyObject_IsTrue(object);
    if (value < 0) throw Raised{};
    return value;
}

int type_code(at::ScalarType type) {
    return type == at::kBFloat16          ? KVSNAP_BF16
           : type == at::kHalf            ? KVSNAP_FP16
           : type == at::kFloat8_e4m3fn   ? KVSNAP_E4M3
           : type == at::kFloat           ? KVSNAP_FP32
                                          : -1;
}

constexpr const char* kTypes[] = {"bfloat16", "float16", "float8_e4m3fn", "float32"};

std::string shape_of(const at::Tensor& t) {
    std::ostringstream text;
    text << t.sizes();
    return text.str();
}

// The calls record nothing for either direction of differentiation: what would be lost is refused.
void check_undifferentiated(const at::Tensor& t, const char* what) {
    if (t.requires_grad() && at::GradMode::is_enabled())
        refuse(what, " requires a gradient, and no gradient is recorded here: call under torch.no_grad()");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        refuse(what, " carries a forward-mode tangent, and none is computed here");
}

// A [tokens, heads, width] tensor (a negative size: any) whose last axis is contiguous.
void check_rows(const at::Tensor& t, const char* what, int64_t tokens, int64_t heads, int64_t width) {
    const auto differs = [&](int axis, int64_t want) { return want >= 0 && t.size(axis) != want; };
    if (t.dim() != 3 || differs(0, tokens) || differs(1, heads) || differs(2, width)) {
        const auto size = [](int64_t n) { return n < 0 ? std::string("any") : std::to_string(n); };
        refuse(what, " must be [", size(tokens), ", ", size(heads), ", ", size(width), "], not ", shape_of(t));
    }
    if (t.stride(2) != 1 && t.size(2) > 1) refuse(what, ": the last axis must be contiguous");
    check_undifferentiated(t, what);
}

void check_device(const at::Device& device, std::initializer_list<const at::Tensor*> tensors) {
    bool same = device.is_cuda();
    for (const at::Tensor* t : tensors) same = same && (!t || t->device() == device);
    if (!same) refuse("every tensor of a call must be on one and the same CUDA device");
}

struct Rotation {
    kvsnap_rotation raw{};
    const at::Tensor* table = nullptr;
    const at::Tensor* positions = nullptr;
};

Rotation rotation_of(PyObject* rotary, PyObject* positions, PyObject* axes, bool interleaved, bool inverse,
                     int64_t tokens, int64_t width) {
    Rotation r;
    if (!given(rotary)) {
        if (given(positions) || given(axes)) refuse("positions and axes need a rotary table");
        return r;
    }
    r.table = &tensor(rotary, "a rotary table");
    if (r.table->dim() != 3 || r.table->size(2) != 2 || r.table->scalar_type() != at::kFloat ||
        !r.table->is_contiguous() || r.table->size(0) == 0)
        refuse("a rotary table is a contiguous float32 [positions, pairs, 2] tensor of one position or more");
    check_undifferentiated(*r.table, "a rotary table");
    const int64_t pairs = r.table->size(1);
    if (pairs == 0 || pairs % 8 || 2 * pairs > width)
        refuse("a rotary table's pairs must be a multiple of 8 and at most ", width / 2, ", not ", pairs);
    int64_t count = 1;
    if (given(positions)) {
        r.positions = &tensor(positions, "positions");
        const at::ScalarType type = r.positions->scalar_type();
        if (type != at::kLong && type != at::kInt) refuse("positions must be int64 or int32");
        const int64_t dims = r.positions->dim();
        if ((dims != 1 && dims != 2) || r.positions->size(-1) != tokens ||
            (r.positions->stride(-1) != 1 && tokens > 1))
            refuse("positions must be [", tokens, "] or [axes, ", tokens, "], the last axis contiguous");
        if (dims == 2) {
            count = r.positions->size(0);
            r.raw.axis_stride = r.positions->stride(0);
        }
        r.raw.positions = r.positions->data_ptr();
        r.raw.narrow = type == at::kInt;
    }
    if (given(axes)) {
        PyObject* const list = PySequence_Fast(axes, "axes must be a sequence of whole numbers");
        if (!list) throw Raised{};
        bool fits = PySequence_Fast_GET_SIZE(list) == pairs && count >= 1 && count <= 4;
        for (int64_t pair = 0; fits && pair < pairs; ++pair) {
            const long axis = PyLong_AsLong(PySequence_Fast_GET_ITEM(list, pair));
            fits = axis >= 0 && axis < count;
            if (fits) r.raw.axes[pair / 8] |= static_cast<uint16_t>(axis << (2 * (pair % 8)));
        }
        Py_DECREF(list);
        if (PyErr_Occurred()) throw Raised{};
        if (!fits)
            refuse("axes must name, for each of ", pairs, " pairs, one of the positions' ", count,
                   " axes (4 at most)");
    } else if (count != 1) {
        refuse("positions of several axes need axes: the axis of each pair");
    }
    r.raw.angles = r.table->data_ptr<float>();
    r.raw.rows = r.table->size(0);
    r.raw.pairs = static_cast<int32_t>(pairs);
    r.raw.interleaved = interleaved;
    r.raw.inverse = inverse;
    return r;
}

struct Sequences {
    kvsnap_sequences raw{};
    const at::Tensor* tables;
    const at::Tensor* lengths;
    const at::Tensor* starts = nullptr;
};

Sequences sequences_of(PyObject* block_tables, PyObject* lengths, PyObject* query_starts, int64_t tokens) {
    Sequences s;
    s.tables = &tensor(block_tables, "block_tables");
    s.lengths = &tensor(lengths, "lengths");
    if (given(query_starts)) s.starts = &tensor(query_starts, "query_starts");
    if (s.tables->dim() != 2 || s.lengths->dim() != 1 || s.tables->size(0) != s.lengths->size(0))
        refuse("block_tables must be [sequences, blocks] and lengths [sequences], not ", shape_of(*s.tables), " and ",
               shape_of(*s.lengths));
    const int64_t count = s.tables->size(0);
    for (const at::Tensor* t : {s.tables, s.lengths, s.starts}) {
        if (!t) continue;
        if (t->scalar_type() != at::kInt) refuse("block_tables, lengths and query_starts must be int32");
        if (t->dim() == 0 || (t->stride(-1) != 1 && t->size(-1) > 1))
            refuse("block_tables, lengths and query_starts must be contiguous along their last axis");
    }
    if (!s.starts && tokens != count)
        refuse(tokens, " rows for ", count, " sequences of one row each: query_starts is needed");
    if (s.starts && (s.starts->dim() != 1 || s.starts->size(0) != count + 1))
        refuse("query_starts must be [", count + 1, "], not ", shape_of(*s.starts));
    if (count >= (int64_t(1) << 30) || s.tables->size(1) >= (int64_t(1) << 30)) refuse("block_tables are too large");
    s.raw.block_tables = s.tables->data_ptr<int32_t>();
    s.raw.lengths = s.lengths->data_ptr<int32_t>();
    s.raw.query_starts = s.starts ? s.starts->data_ptr<int32_t>() : nullptr;
    s.raw.table_stride = s.tables->stride(0);
    s.raw.table_width = static_cast<int32_t>(s.tables->size(1));
    s.raw.n_seqs = static_cast<int32_t>(count);
    return s;
}

// Calls `launch(stream)` with `device` current and Python's lock released; the C entry points' message is the error.
template <typename Launch>
void launched(const at::Device& device, Launch&& launch) {
    const c10::DeviceGuard guard(device);
    const auto stream = reinterpret_cast<uintptr_t>(c10::hip::getCurrentHIPStream(device.index()).stream());
    std::string message;
    Py_BEGIN_ALLOW_THREADS
    if (launch(stream) < 0) message = library.error();
    Py_END_ALLOW_THREADS
    if (!message.empty()) throw std::runtime_error(message);
}

template <typename Call>
PyObject* answered(Py_ssize_t count, Py_ssize_t wanted, Call&& call) {
    try {
        if (count != wanted) throw std::runtime_error("wrong number of arguments");
        return call();
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* const torch = PyImport_ImportModule("torch");
        PyObject* const type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (type) PyErr_SetString(type, e.what());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// An output of `like`'s type: `object` if given, of these sizes.
at::Tensor output(PyObject* object, const char* what, at::IntArrayRef sizes, const at::Tensor& like) {
    if (!given(object)) return at::empty(sizes, like.options().memory_format(at::MemoryFormat::Contiguous));
    const at::Tensor& out = tensor(object, what);
    check_rows(out, what, sizes[0], sizes[1], sizes[2]);
    if (out.scalar_type() != like.scalar_type()) refuse(what, " must have the type of what it holds");
    // Rows and heads apart from one another: the nearer axis by a head's width, the farther by all of the nearer.
    const bool heads_inside = out.stride(1) <= out.stride(0) || out.size(0) <= 1;
    const int inner = heads_inside && out.size(1) > 1 ? 1 : 0, outer = 1 - inner;
    if (out.numel() > 0 && ((out.size(inner) > 1 && out.stride(inner) < out.size(2)) ||
                            (out.size(outer) > 1 && out.stride(outer) < (out.size(inner) - 1) * out.stride(inner) + out.size(2))))
        refuse(what, " must not overlap itself");
    return out;
}

// Whether two [tokens, heads, width] tensors share memory.  Where their ranges meet, they are apart if along an axis of
// one stride each lies in its own part of every period (heads of one projection), or, with both strides alike, in its own
// part of every inner one.
bool meet(const at::Tensor& a, const at::Tensor& b) {
    struct Places {
        int64_t first, size[2], stride[2], width;
        explicit Places(const at::Tensor& t)
            : first(reinterpret_cast<intptr_t>(t.data_ptr())), size{t.size(0), t.size(1)},
              stride{t.stride(0) * t.element_size(), t.stride(1) * t.element_size()},
              width(t.size(2) * t.element_size()) {}
        int64_t extent(int axis) const { return (size[axis] - 1) * stride[axis] + width; }
        int64_t end() const { return first + (size[0] - 1) * stride[0] + extent(1); }
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    const Places x(a), y(b);
    if (x.end() <= y.first || y.end() <= x.first) return false;
    const auto period = [&](int axis) -> int64_t {          // the stride of both, 0 if they differ
        const int64_t of = x.size[axis] > 1 ? x.stride[axis] : y.stride[axis];
        return (x.size[axis] > 1 && x.stride[axis] != of) || (y.size[axis] > 1 && y.stride[axis] != of) ? 0 : of;
    };
    const auto apart = [&](int64_t each, int64_t x_extent, int64_t y_extent) {
        const int64_t at = ((y.first - x.first) % each + each) % each;
        return at >= x_extent && at + y_extent <= each;
    };
    for (const int axis : {0, 1})
        if (period(axis) > 0 && apart(period(axis), x.extent(1 - axis), y.extent(1 - axis))) return false;
    const int64_t outer = std::max(period(0), period(1)), inner = std::min(period(0), period(1));
    return !(inner > 0 && outer % inner == 0 && apart(inner, x.width, y.width));
}

bool same_places(const at::Tensor& a, const at::Tensor& b) {
    bool same = a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes();
    for (int64_t axis = 0; same && axis < a.dim(); ++axis) same = a.size(axis) <= 1 || a.stride(axis) == b.stride(axis);
    return same;
}

// Rows are read while others are written: a given output is the rows it is made from, or apart from them.
void check_apart(PyObject* object, const at::Tensor& out, const char* what, const at::Tensor& from, const char* name,
                 bool itself) {
    if (!given(object) || (itself && same_places(out, from)) || !meet(out, from)) return;
    if (itself) refuse(what, " must be ", name, " itself or not overlap it");
    refuse(what, " must not overlap ", name);
}

// Tells autograd that a tensor's values changed, as torch's own in-place operators do: a graph that saved it must not
// use them.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ----------------------------------------------------------------- calls

// bind(rotate, append, attend, attend_workspace_bytes, cuda_error): the entry points' addresses.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return answered(count, 5, [&]() -> PyObject* {
        const auto at = [&](int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(whole(args[i]))); };
        library.rotate = reinterpret_cast<decltype(library.rotate)>(at(0));
        library.append = reinterpret_cast<decltype(library.append)>(at(1));
        library.attend = reinterpret_cast<decltype(library.attend)>(at(2));
        library.workspace_bytes = reinterpret_cast<decltype(library.workspace_bytes)>(at(3));
        library.error = reinterpret_cast<decltype(library.error)>(at(4));
        Py_RETURN_NONE;
    });
}

// rotate(x, positions, rotary, axes, interleaved, inverse, out)
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return answered(count, 7, [&] {
        const at::Tensor& x = tensor(args[0], "x");
        check_rows(x, "x", -1, -1, -1);
        const int64_t tokens = x.size(0), heads = x.size(1), width = x.size(2);
        const int type = type_code(x.scalar_type());
        if (type < 0 || type == KVSNAP_E4M3) refuse("x must be bfloat16, float16 or float32");
        if (width % 16 || width <= 0 || width > 256)
            refuse("x's width must be a multiple of 16 up to 256, not ", width);
        if (!given(args[1]) || !given(args[2])) refuse("a rotation needs positions and a rotary table");
        const Rotation r = rotation_of(args[2], args[1], args[3], truth(args[4]), truth(args[5]), tokens, width);
        const at::Tensor out = output(args[6], "out", {tokens, heads, width}, x);
        check_apart(args[6], out, "out", x, "x", true);
        check_device(x.device(), {&out, r.table, r.positions});
        launched(x.device(), [&](uintptr_t stream) {
            return library.rotate(x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0),
                                  out.stride(1), tokens, static_cast<int>(heads), static_cast<int>(width), type,
                                  &r.raw, stream);
        });
        if (given(args[6])) written(out);
        return THPVariable_Wrap(out);
    });
}

struct Layer {
    const kvsnap_paged_layer* raw;
    at::Device device;

    Layer(PyObject* address, PyObject* cache)
        : raw(reinterpret_cast<const kvsnap_paged_layer*>(static_cast<uintptr_t>(whole(address)))),
          device(THPVariable_Unpack(cache).device()) {
        check_undifferentiated(THPVariable_Unpack(cache), "the cache");
    }
};

// append(layer, cache, key, value, block_tables, lengths, query_starts, query, positions, rotary, axes, interleaved,
// query_out)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return answered(count, 13, [&]() -> PyObject* {
        const Layer layer(args[0], args[1]);
        const at::Tensor &key = tensor(args[2], "key"), &value = tensor(args[3], "value");
        check_rows(key, "key", -1, layer.raw->kv_heads, layer.raw->width);
        const int64_t tokens = key.size(0), width = layer.raw->width;
        check_rows(value, "value", tokens, layer.raw->kv_heads, width);
        const int type = type_code(key.scalar_type());
        if ((type != KVSNAP_BF16 && type != KVSNAP_FP16) || value.scalar_type() != key.scalar_type() ||
            (layer.raw->type != KVSNAP_E4M3 && layer.raw->type != type))
            refuse("keys and values must both be bfloat16 or float16, a 16-bit cache's own type: ",
                   key.scalar_type(), " and ", value.scalar_type(), " into ", kTypes[layer.raw->type]);
        const Sequences s = sequences_of(args[4], args[5], args[6], tokens);
        const Rotation r = rotation_of(args[9], args[8], args[10], truth(args[11]), false, tokens, width);
        at::Tensor out;
        const at::Tensor* query = nullptr;
        if (given(args[7])) {
            query = &tensor(args[7], "query");
            check_rows(*query, "query", tokens, -1, width);
            if (query->scalar_type() != key.scalar_type()) refuse("query must have the keys' type");
            out = output(args[12], "query_out", query->sizes(), *query);
            check_apart(args[12], out, "query_out", *query, "query", true);
            check_apart(args[12], out, "query_out", key, "key", false);
            check_apart(args[12], out, "query_out", value, "value", false);
        } else if (given(args[12])) {
            refuse("query_out needs a query");
        }
        check_device(layer.device, {&key, &value, s.tables, s.lengths, s.starts, query, query ? &out : nullptr,
                                    r.table, r.positions});
        launched(layer.device, [&](uintptr_t stream) {
            return library.append(layer.raw, &s.raw, &r.raw, key.data_ptr(), key.stride(0), key.stride(1),
                                  value.data_ptr(), value.stride(0), value.stride(1),
                                  query ? query->data_ptr() : nullptr, query ? query->stride(0) : 0,
                                  query ? query->stride(1) : 0, query ? out.data_ptr() : nullptr,
                                  query ? out.stride(0) : 0, query ? out.stride(1) : 0, tokens,
                                  query ? static_cast<int>(query->size(1)) : 0, type, stream);
        });
        written(THPVariable_Unpack(args[1]));
        if (given(args[12])) written(out);
        if (!query) Py_RETURN_NONE;
        return THPVariable_Wrap(out);
    });
}

// attend(layer, cache, query, block_tables, lengths, query_starts, max_length, softmax_scale, window, out,
// return_lse)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return answered(count, 11, [&]() -> PyObject* {
        const Layer layer(args[0], args[1]);
        const int64_t kv_heads = layer.raw->kv_heads, width = layer.raw->width;
        const at::Tensor& query = tensor(args[2], "query");
        check_rows(query, "query", -1, -1, width);
        const int64_t tokens = query.size(0), heads = query.size(1);
        const int type = type_code(query.scalar_type());
        if ((type != KVSNAP_BF16 && type != KVSNAP_FP16) ||
            (layer.raw->type != KVSNAP_E4M3 && layer.raw->type != type))
            refuse("queries must be bfloat16 or float16, a 16-bit cache's own type: ", query.scalar_type(), " over ",
                   kTypes[layer.raw->type]);
        if (heads == 0 || heads % kv_heads) refuse(heads, " query heads do not share the cache's ", kv_heads);
        double scale = 1.0 / std::sqrt(static_cast<double>(width));
        if (given(args[7])) {
            scale = PyFloat_AsDouble(args[7]);
            if (scale == -1.0 && PyErr_Occurred()) throw Raised{};
        }
        if (!(scale > 0) || !(scale < 1e30)) refuse("softmax_scale must be positive and finite");
        int64_t window = 0;
        if (given(args[8])) {
            window = whole(args[8]);
            if (window < 1) refuse("a window holds at least the row's own token");
            window = std::min(window, int64_t(1) << 30);
        }
        const Sequences s = sequences_of(args[3], args[4], args[5], tokens);
        const int64_t named = s.tables->size(1) * layer.raw->block_size;
        int64_t longest = named;
        if (given(args[6])) {
            longest = std::min(longest, whole(args[6]));
            if (longest < 0) refuse("max_length must not be negative");
        }
        const at::Tensor out = output(args[9], "out", query.sizes(), query);
        check_apart(args[9], out, "out", query, "query", true);
        const bool wants_lse = truth(args[10]);
        check_device(layer.device, {&query, &out, s.tables, s.lengths, s.starts});
        at::Tensor lse, scratch;
        if (wants_lse) lse = at::empty({tokens, heads}, query.options().dtype(at::kFloat));
        const size_t size = library.workspace_bytes(layer.raw, tokens, s.raw.n_seqs, s.starts != nullptr,
                                                    static_cast<int>(heads), longest, window);
        if (size) scratch = at::empty({static_cast<int64_t>(size)}, query.options().dtype(at::kByte));
        launched(layer.device, [&](uintptr_t stream) {
            return library.attend(layer.raw, &s.raw, query.data_ptr(), query.stride(0), query.stride(1),
                                  out.data_ptr(), out.stride(0), out.stride(1),
                                  wants_lse ? lse.data_ptr<float>() : nullptr, tokens, static_cast<int>(heads), type,
                                  static_cast<float>(scale), window, longest, size ? scratch.data_ptr() : nullptr,
                                  size, stream);
        });
        if (given(args[9])) written(out);
        if (!wants_lse) return THPVariable_Wrap(out);
        PyObject* const first = THPVariable_Wrap(out);
        PyObject* const second = THPVariable_Wrap(lse);
        return Py_BuildValue("(NN)", first, second);
    });
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(rotate), FAST(append), FAST(attend), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kvsnap_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kvsnap_binding() { return PyModule_Create(&module); }
