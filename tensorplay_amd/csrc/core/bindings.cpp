// Python bindings (pybind11; nanobind, which the reference uses, is not in this
// image).  The method overloads mirror TensorPlay's reduction surface
// (/root/reference/src/bindings/python/Tensor.cpp:1099-1224): each reduction
// takes dim as an int or a list, keepdim, and (sum/mean) a keyword dtype;
// var/std take correction.  topk is added.  C++ exceptions map to the Python
// exception of the same name (as src/bindings/python/init.cpp:13-38).
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <sstream>

#include "Allocator.h"
#include "Dispatcher.h"
#include "Exception.h"
#include "FineTune.h"
#include "Tensor.h"
#include "tpr_rocm.h"

namespace py = pybind11;
using namespace tensorplay;

namespace {

DType dtype_from_numpy(const py::dtype& dt) {
    const char k = dt.kind();
    const size_t sz = dt.itemsize();
    if (k == 'f' && sz == 2) return DType::Float16;
    if (k == 'f' && sz == 4) return DType::Float32;
    if (k == 'f' && sz == 8) return DType::Float64;
    if (k == 'i' && sz == 8) return DType::Int64;
    if (k == 'i' && sz == 4) return DType::Int32;
    if (k == 'i' && sz == 2) return DType::Int16;
    if (k == 'i' && sz == 1) return DType::Int8;
    if (k == 'u' && sz == 1) return DType::UInt8;
    if (k == 'u' && sz == 2) return DType::UInt16;
    if (k == 'u' && sz == 4) return DType::UInt32;
    if (k == 'u' && sz == 8) return DType::UInt64;
    if (k == 'b') return DType::Bool;
    TP_THROW(TypeError, "unsupported numpy dtype");
}

py::dtype numpy_dtype(DType t) {
    switch (t) {
        case DType::Float32: return py::dtype::of<float>();
        case DType::Float64: return py::dtype::of<double>();
        case DType::Int64: return py::dtype::of<int64_t>();
        case DType::Int32: return py::dtype::of<int32_t>();
        case DType::Int16: return py::dtype::of<int16_t>();
        case DType::Int8: return py::dtype::of<int8_t>();
        case DType::UInt8: return py::dtype::of<uint8_t>();
        case DType::UInt16: return py::dtype::of<uint16_t>();
        case DType::UInt32: return py::dtype::of<uint32_t>();
        case DType::UInt64: return py::dtype::of<uint64_t>();
        case DType::Bool: return py::dtype::of<bool>();
        case DType::Float16: return py::dtype("float16");
        default: TP_THROW(TypeError, "no numpy dtype for this tensor dtype");
    }
}

Device to_device(const py::object& o) {
    if (py::isinstance<Device>(o)) return o.cast<Device>();
    return Device(o.cast<std::string>());
}

Tensor from_numpy(py::array arr, std::optional<DType> dtype, const py::object& device) {
    py::array c = py::array::ensure(arr, py::array::c_style | py::array::forcecast);
    DType dt = dtype_from_numpy(c.dtype());
    if (dtype && *dtype != dt) {
        c = py::array(numpy_dtype(*dtype), py::array::ShapeContainer(c.shape(), c.shape() + c.ndim()));
        py::array src = py::array::ensure(arr, py::array::c_style | py::array::forcecast);
        py::module_::import("numpy").attr("copyto")(c, src, py::arg("casting") = "unsafe");
        dt = *dtype;
    }
    std::vector<int64_t> shape(c.shape(), c.shape() + c.ndim());
    return Tensor::fromHost(c.data(), shape, dt, to_device(device));
}

py::array to_numpy(const Tensor& t) {
    std::vector<py::ssize_t> shape(t.shape().begin(), t.shape().end());
    py::array out(numpy_dtype(t.dtype()), shape);
    t.copyToHost(out.mutable_data());
    return out;
}

// Keeps a Python object alive for as long as a tensor views its memory; the last
// reference may go on any thread.
std::shared_ptr<void> hold(PyObject* o) {
    Py_INCREF(o);
    return std::shared_ptr<void>(o, [](void* p) {
        if (PyGILState_Check()) {
            Py_DECREF(static_cast<PyObject*>(p));
        } else {
            py::gil_scoped_acquire g;
            Py_DECREF(static_cast<PyObject*>(p));
        }
    });
}

py::object steal(PyObject* o) {
    if (!o) throw py::error_already_set();
    return py::reinterpret_steal<py::object>(o);
}

int64_t whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
    return v;
}

std::vector<int64_t> extents(const py::object& t) {
    if (!PyTuple_Check(t.ptr())) return t.cast<std::vector<int64_t>>();
    std::vector<int64_t> v(PyTuple_GET_SIZE(t.ptr()));
    for (size_t i = 0; i < v.size(); ++i) v[i] = whole(PyTuple_GET_ITEM(t.ptr(), i));
    return v;
}

// torch's element types and the names of a tensor's members, looked up once
struct TorchNames {
    std::vector<std::pair<PyObject*, DType>> types;
    PyObject *is_cuda, *dtype, *data_ptr, *shape, *stride, *get_device;
    TorchNames() {
        const py::module_ torch = py::module_::import("torch");
        for (const auto& [name, dt] : std::initializer_list<std::pair<const char*, DType>>{
                 {"float32", DType::Float32}, {"bfloat16", DType::BFloat16}, {"float16", DType::Float16},
                 {"int64", DType::Int64}, {"float64", DType::Float64}, {"int32", DType::Int32}, {"int16", DType::Int16},
                 {"int8", DType::Int8}, {"uint8", DType::UInt8}, {"bool", DType::Bool}})
            types.emplace_back(py::object(torch.attr(name)).release().ptr(), dt);
        is_cuda = PyUnicode_InternFromString("is_cuda");
        dtype = PyUnicode_InternFromString("dtype");
        data_ptr = PyUnicode_InternFromString("data_ptr");
        shape = PyUnicode_InternFromString("shape");
        stride = PyUnicode_InternFromString("stride");
        get_device = PyUnicode_InternFromString("get_device");
    }
};

// A torch tensor's memory as a Tensor: zero-copy on an AMD GPU, a copy on the host.
Tensor from_torch(const py::object& o) {
    // The interpreter's lock orders this, and no lock of its own: a thread that waited for a
    // guarded initialization would hold the lock that the import may have let go of.  Two
    // threads may both look the names up; one set is kept.
    static const TorchNames* names = nullptr;
    if (!names) names = new TorchNames();
    const TorchNames* const n = names;
    PyObject* t = o.ptr();
    if (steal(PyObject_GetAttr(t, n->is_cuda)).ptr() != Py_True)
        return from_numpy(py::array(o.attr("detach")().attr("numpy")()), std::nullopt, py::str("cpu"));
    const py::object dtype = steal(PyObject_GetAttr(t, n->dtype));
    for (const auto& [type, dt] : n->types) {
        if (type != dtype.ptr()) continue;
        const int64_t p = whole(steal(PyObject_CallMethodNoArgs(t, n->data_ptr)).ptr());
        const int64_t dev = whole(steal(PyObject_CallMethodNoArgs(t, n->get_device)).ptr());
        return Tensor::fromExternal(reinterpret_cast<void*>((uintptr_t)p), extents(steal(PyObject_GetAttr(t, n->shape))),
                                    extents(steal(PyObject_CallMethodNoArgs(t, n->stride))), dt,
                                    Device(DeviceType::ROCm, (int)dev), hold(t));
    }
    throw py::key_error(py::str(dtype).cast<std::string>());
}

// DLPack's structures (the unversioned ABI of its specification).
struct DLTensor {
    void* data;
    int32_t device_type, device_id;
    int32_t ndim;
    uint8_t code, bits;
    uint16_t lanes;
    int64_t* shape;
    int64_t* strides;
    uint64_t byte_offset;
};
struct DLManagedTensor {
    DLTensor tensor;
    void* ctx;
    void (*deleter)(DLManagedTensor*);
};
struct DLHolder {
    DLManagedTensor dl;
    Tensor owner;
    std::vector<int64_t> shape, strides;
};

py::capsule to_dlpack(const Tensor& t) {
    auto h = std::make_unique<DLHolder>();
    h->owner = t;
    h->shape = t.shape();
    h->strides = t.strides();
    DLTensor& d = h->dl.tensor;
    d.data = t.data_ptr();
    d.device_type = t.device().is_cpu() ? 1 : 10;  // kDLCPU, kDLROCM
    d.device_id = t.device().is_cpu() ? 0 : t.device().index;
    d.ndim = (int32_t)t.dim();
    switch (t.dtype()) {
        case DType::Float16: case DType::Float32: case DType::Float64: d.code = 2; break;
        case DType::BFloat16: d.code = 4; break;
        case DType::Bool: d.code = 6; break;
        case DType::UInt8: case DType::UInt16: case DType::UInt32: case DType::UInt64: d.code = 1; break;
        default: d.code = 0;
    }
    d.bits = (uint8_t)(8 * t.element_size());
    d.lanes = 1;
    d.shape = h->shape.data();
    d.strides = h->strides.data();
    d.byte_offset = 0;
    h->dl.ctx = h.get();
    h->dl.deleter = [](DLManagedTensor* m) { delete static_cast<DLHolder*>(m->ctx); };
    PyObject* c = PyCapsule_New(&h->dl, "dltensor", [](PyObject* o) {
        if (!PyCapsule_IsValid(o, "dltensor")) return;  // taken over by its consumer
        auto* m = static_cast<DLManagedTensor*>(PyCapsule_GetPointer(o, "dltensor"));
        m->deleter(m);
    });
    if (!c) throw py::error_already_set();
    h.release();
    return py::reinterpret_steal<py::capsule>(c);
}

std::string repr(const Tensor& t) {
    std::ostringstream os;
    os << "tensor(shape=[";
    for (size_t i = 0; i < t.shape().size(); ++i) os << (i ? ", " : "") << t.shape()[i];
    os << "], dtype=" << toString(t.dtype()) << ", device=" << t.device().str() << ")";
    return os.str();
}

DType opt_dtype(const std::optional<DType>& d) { return d.value_or(DType::Undefined); }

}  // namespace

PYBIND11_MODULE(_C, m) {
    m.doc() = "tensorplay_amd native core: P10-shaped tensor + dispatcher with a ROCm backend";

    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const IndexError& e) {
            PyErr_SetString(PyExc_IndexError, e.what());
        } catch (const TypeError& e) {
            PyErr_SetString(PyExc_TypeError, e.what());
        } catch (const ValueError& e) {
            PyErr_SetString(PyExc_ValueError, e.what());
        } catch (const NotImplementedError& e) {
            PyErr_SetString(PyExc_NotImplementedError, e.what());
        } catch (const RuntimeError& e) {
            PyErr_SetString(PyExc_RuntimeError, e.what());
        }
    });

    py::enum_<DType>(m, "DType")
        .value("uint8", DType::UInt8).value("int8", DType::Int8).value("int16", DType::Int16)
        .value("int32", DType::Int32).value("int64", DType::Int64).value("uint16", DType::UInt16)
        .value("uint32", DType::UInt32).value("uint64", DType::UInt64).value("float32", DType::Float32)
        .value("float64", DType::Float64).value("bool", DType::Bool).value("undefined", DType::Undefined)
        .value("float16", DType::Float16).value("bfloat16", DType::BFloat16);

    py::class_<Device>(m, "Device")
        .def(py::init<const std::string&>())
        .def_property_readonly("type", [](const Device& d) { return d.is_cpu() ? "cpu" : "rocm"; })
        .def_property_readonly("index", [](const Device& d) { return d.index; })
        .def("__repr__", [](const Device& d) { return "device('" + d.str() + "')"; })
        .def("__str__", &Device::str)
        .def("__eq__", [](const Device& a, const Device& b) { return a == b; });

    py::class_<Tensor> t(m, "TensorBase");
    t.def_property_readonly("shape", [](const Tensor& x) { return std::vector<int64_t>(x.shape()); })
        .def_property_readonly("dtype", &Tensor::dtype)
        .def_property_readonly("device", &Tensor::device)
        .def_property_readonly("ndim", &Tensor::dim)
        .def("dim", &Tensor::dim)
        .def("numel", &Tensor::numel)
        .def("size", [](const Tensor& x, std::optional<int64_t> d) -> py::object {
            if (d) return py::int_(x.size(*d));
            return py::cast(std::vector<int64_t>(x.shape()));
        }, py::arg("dim") = py::none())
        .def("stride", [](const Tensor& x) { return std::vector<int64_t>(x.strides()); })
        .def("storage_offset", &Tensor::storage_offset)
        .def("is_contiguous", &Tensor::is_contiguous)
        .def("contiguous", &Tensor::contiguous)
        .def("clone", &Tensor::clone)
        .def("data_ptr", [](const Tensor& x) { return reinterpret_cast<uintptr_t>(x.data_ptr()); })
        .def("record_stream", [](const Tensor& x, uintptr_t s) { x.record_stream(reinterpret_cast<void*>(s)); },
             py::arg("stream"))
        .def("transpose", &Tensor::transpose)
        .def("permute", [](const Tensor& x, const std::vector<int64_t>& d) { return x.permute(d); })
        .def("reshape", [](const Tensor& x, const std::vector<int64_t>& s) { return x.reshape(s); })
        .def("to", [](const Tensor& x, const py::object& arg) {
            if (py::isinstance<DType>(arg)) return x.to(arg.cast<DType>());
            return x.to(to_device(arg));
        })
        .def("copy_", [](Tensor& x, const Tensor& src) { return x.copy_(src); }, py::arg("src"))
        .def("cpu", &Tensor::cpu)
        .def("rocm", [](const Tensor& x, int index) { return x.to(Device(DeviceType::ROCm, index)); },
             py::arg("index") = 0)
        .def("numpy", &to_numpy)
        .def("item", [](const Tensor& x) -> py::object {
            if (isIntegralType(x.dtype(), false)) return py::int_(x.item_int());
            if (x.dtype() == DType::Bool) return py::bool_(x.item() != 0.0);
            return py::float_(x.item());
        })
        .def("__repr__", &repr)
        .def("__getitem__", [](const Tensor& x, int64_t i) {
            if (x.dim() == 0) TP_THROW(IndexError, "invalid index of a 0-dim tensor");
            const int64_t n = x.shape()[0];
            if (i < 0) i += n;
            if (i < 0 || i >= n) TP_THROW(IndexError, "index out of range");
            std::vector<int64_t> sz(x.shape().begin() + 1, x.shape().end());
            std::vector<int64_t> st(x.strides().begin() + 1, x.strides().end());
            return x.as_strided(sz, st, x.storage_offset() + i * x.strides()[0]);
        });

    // ---- reductions (Tensor.cpp:1101-1224 overload set) ----
    using V = std::vector<int64_t>;
    t.def("sum", [](const Tensor& s, std::optional<DType> dt) { return s.sum(opt_dtype(dt)); },
          py::kw_only(), py::arg("dtype") = py::none())
        .def("sum", [](const Tensor& s, const V& d, bool k, std::optional<DType> dt) { return s.sum(d, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("sum", [](const Tensor& s, int64_t d, bool k, std::optional<DType> dt) { return s.sum(V{d}, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("mean", [](const Tensor& s, std::optional<DType> dt) { return s.mean(opt_dtype(dt)); },
             py::kw_only(), py::arg("dtype") = py::none())
        .def("mean", [](const Tensor& s, const V& d, bool k, std::optional<DType> dt) { return s.mean(d, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("mean", [](const Tensor& s, int64_t d, bool k, std::optional<DType> dt) { return s.mean(V{d}, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("max", [](const Tensor& s) { return s.max(); })
        .def("max", [](const Tensor& s, const V& d, bool k) { return s.max(d, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("max", [](const Tensor& s, int64_t d, bool k) { return s.max(V{d}, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("min", [](const Tensor& s) { return s.min(); })
        .def("min", [](const Tensor& s, const V& d, bool k) { return s.min(d, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("min", [](const Tensor& s, int64_t d, bool k) { return s.min(V{d}, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("argmax", [](const Tensor& s, std::optional<int64_t> d, bool k) { return s.argmax(d, k); },
             py::arg("dim") = py::none(), py::arg("keepdim") = false)
        .def("argmin", [](const Tensor& s, std::optional<int64_t> d, bool k) { return s.argmin(d, k); },
             py::arg("dim") = py::none(), py::arg("keepdim") = false)
        .def("var", [](const Tensor& s, int64_t c) { return s.var(c); }, py::arg("correction") = 1)
        .def("var", [](const Tensor& s, const V& d, int64_t c, bool k) { return s.var(d, c, k); }, py::arg("dim"),
             py::arg("correction") = 1, py::arg("keepdim") = false)
        .def("var", [](const Tensor& s, int64_t d, int64_t c, bool k) { return s.var(V{d}, c, k); }, py::arg("dim"),
             py::arg("correction") = 1, py::arg("keepdim") = false)
        .def("std", [](const Tensor& s, int64_t c) { return s.std(c); }, py::arg("correction") = 1)
        .def("std", [](const Tensor& s, const V& d, int64_t c, bool k) { return s.std(d, c, k); }, py::arg("dim"),
             py::arg("correction") = 1, py::arg("keepdim") = false)
        .def("std", [](const Tensor& s, int64_t d, int64_t c, bool k) { return s.std(V{d}, c, k); }, py::arg("dim"),
             py::arg("correction") = 1, py::arg("keepdim") = false)
        .def("prod", [](const Tensor& s, std::optional<DType> dt) { return s.prod(opt_dtype(dt)); },
             py::kw_only(), py::arg("dtype") = py::none())
        .def("prod", [](const Tensor& s, const V& d, bool k, std::optional<DType> dt) { return s.prod(d, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("prod", [](const Tensor& s, int64_t d, bool k, std::optional<DType> dt) { return s.prod(V{d}, k, opt_dtype(dt)); },
             py::arg("dim"), py::arg("keepdim") = false, py::kw_only(), py::arg("dtype") = py::none())
        .def("all", [](const Tensor& s) { return s.all(); })
        .def("all", [](const Tensor& s, const V& d, bool k) { return s.all(d, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("all", [](const Tensor& s, int64_t d, bool k) { return s.all(V{d}, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("any", [](const Tensor& s) { return s.any(); })
        .def("any", [](const Tensor& s, const V& d, bool k) { return s.any(d, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("any", [](const Tensor& s, int64_t d, bool k) { return s.any(V{d}, k); }, py::arg("dim"),
             py::arg("keepdim") = false)
        .def("median", [](const Tensor& s) { return s.median(); })
        .def("norm", [](const Tensor& s, double p) { return s.norm(p); }, py::arg("p") = 2.0)
        .def("norm", [](const Tensor& s, const V& d, double p, bool k) { return s.norm(d, p, k); }, py::arg("dim"),
             py::arg("p") = 2.0, py::arg("keepdim") = false)
        .def("norm", [](const Tensor& s, int64_t d, double p, bool k) { return s.norm(V{d}, p, k); }, py::arg("dim"),
             py::arg("p") = 2.0, py::arg("keepdim") = false)
        .def("topk", [](const Tensor& s, int64_t k, int64_t d, bool largest, bool sorted) {
            return s.topk(k, d, largest, sorted);
        }, py::arg("k"), py::arg("dim") = -1, py::arg("largest") = true, py::arg("sorted") = true)
        .def("softmax", [](const Tensor& s, int64_t d, std::optional<DType> dt) { return s.softmax(d, opt_dtype(dt)); },
             py::arg("dim"), py::arg("dtype") = py::none())
        .def("log_softmax", [](const Tensor& s, int64_t d, std::optional<DType> dt) {
            return s.log_softmax(d, opt_dtype(dt));
        }, py::arg("dim"), py::arg("dtype") = py::none());

    // ---- function-only schemas (tensorplay/functional.py:313-317, 496-500) ----
    m.def("softmax", [](const Tensor& s, int64_t d, std::optional<DType> dt) { return s.softmax(d, opt_dtype(dt)); },
          py::arg("self"), py::arg("dim"), py::arg("dtype") = py::none());
    m.def("log_softmax", [](const Tensor& s, int64_t d, std::optional<DType> dt) {
        return s.log_softmax(d, opt_dtype(dt));
    }, py::arg("self"), py::arg("dim"), py::arg("dtype") = py::none());
    m.def("nll_loss", [](const Tensor& s, const Tensor& t, std::optional<Tensor> w, int64_t r, int64_t ig) {
        return nll_loss(s, t, w, r, ig);
    }, py::arg("self"), py::arg("target"), py::arg("weight") = py::none(), py::arg("reduction") = 1,
       py::arg("ignore_index") = -100);
    m.def("nll_loss_backward", [](const Tensor& g, const Tensor& s, const Tensor& t, std::optional<Tensor> w,
                                  int64_t r, int64_t ig, std::optional<Tensor> tw) {
        return nll_loss_backward(g, s, t, w, r, ig, tw.value_or(Tensor()));
    }, py::arg("grad_output"), py::arg("self"), py::arg("target"), py::arg("weight") = py::none(),
       py::arg("reduction") = 1, py::arg("ignore_index") = -100, py::arg("total_weight") = py::none());
    m.def("topk_topp_sample", [](const Tensor& s, const Tensor& u, int64_t k, double t, double p) {
        return topk_topp_sample(s, u, k, t, p);
    }, py::arg("self"), py::arg("uniforms"), py::arg("k") = 50, py::arg("temperature") = 1.0, py::arg("top_p") = 1.0);
    m.def("sum_backward", [](const Tensor& g, const Tensor& s, const V& d, bool k) { return sum_backward(g, s, d, k); },
          py::arg("grad"), py::arg("self"), py::arg("dim") = V{}, py::arg("keepdim") = false);
    m.def("mean_backward", [](const Tensor& g, const Tensor& s, const V& d, bool k) { return mean_backward(g, s, d, k); },
          py::arg("grad"), py::arg("self"), py::arg("dim") = V{}, py::arg("keepdim") = false);
    m.def("var_backward", [](const Tensor& g, const Tensor& s, const V& d, int64_t c, bool k) {
        return var_backward(g, s, d, c, k);
    }, py::arg("grad"), py::arg("self"), py::arg("dim") = V{}, py::arg("correction") = 1, py::arg("keepdim") = false);
    m.def("std_backward", [](const Tensor& g, const Tensor& s, const Tensor& r, const V& d, int64_t c, bool k) {
        return std_backward(g, s, r, d, c, k);
    }, py::arg("grad"), py::arg("self"), py::arg("result"), py::arg("dim") = V{}, py::arg("correction") = 1,
       py::arg("keepdim") = false);
    m.def("_softmax_backward_data", [](const Tensor& g, const Tensor& y, int64_t d) {
        return _softmax_backward_data(g, y, d, DType::Float32);
    }, py::arg("grad_output"), py::arg("output"), py::arg("dim"));
    m.def("_log_softmax_backward_data", [](const Tensor& g, const Tensor& y, int64_t d) {
        return _log_softmax_backward_data(g, y, d, DType::Float32);
    }, py::arg("grad_output"), py::arg("output"), py::arg("dim"));

    // ---- operators of a fine-tuning step (FineTune.h) ----
    using T = const Tensor&;
    using O = std::optional<Tensor>;
    m.def("token_logprob", &token_logprob, py::arg("self"), py::arg("target"), py::arg("temperature") = 1.0,
          py::arg("ignore_index") = -100);
    m.def("token_logprob_backward", &token_logprob_backward, py::arg("grad"), py::arg("self"), py::arg("target"),
          py::arg("lse"), py::arg("temperature") = 1.0, py::arg("ignore_index") = -100);
    m.def("policy_loss", &policy_loss, py::arg("self"), py::arg("target"), py::arg("old_logp"), py::arg("advantage"),
          py::arg("ref_logp") = py::none(), py::arg("weight") = py::none(), py::arg("clip_low") = 0.2,
          py::arg("clip_high") = 0.2, py::arg("kl_coef") = 0.0, py::arg("temperature") = 1.0,
          py::arg("ignore_index") = -100);
    m.def("policy_loss_and_grad", &policy_loss_and_grad, py::arg("self"), py::arg("target"), py::arg("old_logp"),
          py::arg("advantage"), py::arg("ref_logp") = py::none(), py::arg("weight") = py::none(),
          py::arg("clip_low") = 0.2, py::arg("clip_high") = 0.2, py::arg("kl_coef") = 0.0, py::arg("temperature") = 1.0,
          py::arg("ignore_index") = -100);
    m.def("policy_loss_backward", &policy_loss_backward, py::arg("grad"), py::arg("coef"), py::arg("self"),
          py::arg("target"), py::arg("lse"), py::arg("temperature") = 1.0, py::arg("ignore_index") = -100);
    m.def("preference_loss", &preference_loss, py::arg("self"), py::arg("target"), py::arg("offsets"),
          py::arg("ref_logp"), py::arg("beta") = 0.1, py::arg("label_smoothing") = 0.0, py::arg("ignore_index") = -100);
    m.def("preference_loss_backward", [](T g, T c, T s, T t, T l, int64_t ig) {
        return preference_loss_backward(g, c, s, t, l, ig);
    }, py::arg("grad"), py::arg("coef"), py::arg("self"), py::arg("target"), py::arg("lse"),
       py::arg("ignore_index") = -100);
    m.def("dropout", &dropout, py::arg("self"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0);
    m.def("dropout_backward", &dropout_backward, py::arg("grad"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0);
    m.def("gated_residual_norm", [](T x, T h, T pre, double eps, O post, O gate, double scale, double p, int64_t seed,
                                    int64_t offset) {
        return gated_residual_norm(x, h, pre, eps, post, gate, scale, p, seed, offset);
    }, py::arg("self"), py::arg("residual"), py::arg("pre_weight"), py::arg("eps") = 1e-6,
       py::arg("post_weight") = py::none(), py::arg("gate") = py::none(), py::arg("residual_scale") = 1.0,
       py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0);
    m.def("gated_residual_norm_backward", [](T gy, O go, T x, T out, O rpost, T rpre, T pre, O post, O gate,
                                             double scale, double p, int64_t seed, int64_t offset) {
        return gated_residual_norm_backward(gy, go, x, out, rpost, rpre, pre, post, gate, scale, p, seed, offset);
    }, py::arg("grad_y"), py::arg("grad_residual"), py::arg("self"), py::arg("out"), py::arg("rstd_post"),
       py::arg("rstd_pre"), py::arg("pre_weight"), py::arg("post_weight") = py::none(), py::arg("gate") = py::none(),
       py::arg("residual_scale") = 1.0, py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0);

    // ---- factories ----
    m.def("tensor", &from_numpy, py::arg("data"), py::arg("dtype") = py::none(), py::arg("device") = "cpu");
    m.def("empty", [](const V& shape, DType dt, const py::object& dev) { return Tensor::empty(shape, dt, to_device(dev)); },
          py::arg("shape"), py::arg("dtype") = DType::Float32, py::arg("device") = "cpu");
    m.def("_from_device_ptr", [](uintptr_t ptr, const V& shape, const V& strides, DType dt, int index, py::object owner) {
        return Tensor::fromExternal(reinterpret_cast<void*>(ptr), shape, strides, dt, Device(DeviceType::ROCm, index),
                                    hold(owner.ptr()));
    }, py::arg("ptr"), py::arg("shape"), py::arg("strides"), py::arg("dtype"), py::arg("device_index"), py::arg("owner"),
       "Wraps device memory owned by `owner` (e.g. a torch tensor) without copying.");
    m.def("_reduction_shape", &reductionShape);
    m.def("_registered_ops", [](const std::string& key, const std::string& ns) {
        if (key == "ROCm") return Dispatcher::singleton().registeredOps(DispatchKey::ROCm, ns);
        if (key == "CPU") return Dispatcher::singleton().registeredOps(DispatchKey::CPU, ns);
        TP_THROW(ValueError, "unknown dispatch key " + key);
    }, py::arg("key"), py::arg("ns") = "");
    m.def("_from_torch", &from_torch, py::arg("t"));
    m.def("_to_dlpack", &to_dlpack, py::arg("self"), "A DLPack capsule over the tensor's memory (no copy).");

    auto r = m.def_submodule("_rocm", "ROCm device runtime");
    r.def("is_available", [] { return rocmDeviceCount() > 0; });
    r.def("device_count", &rocmDeviceCount);
    r.def("synchronize", &synchronize, py::arg("device") = 0);
    r.def("set_stream", [](uintptr_t s, int dev) { setCurrentStream(dev, reinterpret_cast<void*>(s)); },
          py::arg("stream"), py::arg("device") = 0);
    r.def("current_stream", [](int dev) { return reinterpret_cast<uintptr_t>(currentStream(dev)); },
          py::arg("device") = 0);
    r.def("empty_cache", &emptyCache);
    r.def("release_stream_blocks", [](uintptr_t s, int dev) { releaseStreamBlocks(dev, reinterpret_cast<void*>(s)); },
          py::arg("stream"), py::arg("device") = 0);
    r.def("memory_stats", [](int dev) {
        AllocatorStats s = allocatorStats(dev);
        py::dict d;
        d["allocated_bytes"] = s.allocated_bytes;
        d["cached_bytes"] = s.cached_bytes;
        d["pending_bytes"] = s.pending_bytes;
        d["device_allocs"] = s.device_allocs;
        d["requests"] = s.requests;
        d["leaked_bytes"] = s.leaked_bytes;
        return d;
    }, py::arg("device") = 0);
    r.def("abi_version", [] { return tpr_abi_version(); });
}
