// Host side of ops.clip_grads: checks a list of gradient tensors and reads their addresses, sizes and types in one call.  In Python the five
// attributes of each of a few hundred tensors cost more than the kernels take (152 tensors: 190 us of attributes against 55 us).
//
//   clip_table(tensors, out, device) -> (src, dst, numel, types) as bytes objects of int64 / int64 / int64 / int32; dst is None without out
//   tensors, out: lists of tensors; out may be None, or the same list for clipping in place; device: index of the current GPU
// Raises ValueError with the reason.  No state is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

static int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

static const at::Tensor& tensor_at(PyObject* list, Py_ssize_t i, const char* what) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) throw std::string(what) + "[" + std::to_string(i) + "]: expected a tensor";
    return THPVariable_Unpack(o);
}

static void check_one(const at::Tensor& t, Py_ssize_t i, const char* what, long device) {
    const std::string name = std::string(what) + "[" + std::to_string(i) + "]";
    if (!t.is_cuda()) throw name + ": expected a GPU tensor (the HIP kernels are the only implementation), got " + t.device().str();
    if (device >= 0 && t.get_device() != device)
        throw name + ": the tensor is on " + t.device().str() + ", the current device is cuda:" + std::to_string(device);
    if (t.layout() != at::kStrided) throw name + ": expected a dense tensor";
    if (type_code(t) < 0) throw name + ": expected float32, bfloat16 or float16, got " + std::string(at::toString(t.scalar_type()));
    if (t.is_neg()) throw name + ": expected the values themselves, not a lazily negated view (resolve_neg)";
    if (!t.is_non_overlapping_and_dense()) throw name + ": expected a dense tensor (every element of its memory range, once)";
}

static PyObject* clip_table(PyObject*, PyObject* args) {
    PyObject *list, *out;
    long device;
    if (!PyArg_ParseTuple(args, "O!Ol", &PyList_Type, &list, &out, &device)) return nullptr;
    if (out != Py_None && !PyList_Check(out)) {
        PyErr_SetString(PyExc_TypeError, "clip_table: out must be a list or None");
        return nullptr;
    }
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        std::vector<int64_t> src(n), dst(n), numel(n);
        std::vector<int32_t> types(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            const at::Tensor& t = tensor_at(list, i, "tensors");
            check_one(t, i, "tensors", device);
            numel[i] = t.numel();
            types[i] = type_code(t);
        }
        if (out != Py_None) {
            if (PyList_GET_SIZE(out) != n) throw std::to_string(n) + " tensors, " + std::to_string(PyList_GET_SIZE(out)) + " outputs";
            for (Py_ssize_t i = 0; i < n; ++i) {
                const at::Tensor& t = tensor_at(list, i, "tensors");
                const at::Tensor& o = tensor_at(out, i, "out");
                if (out != list) {
                    check_one(o, i, "out", device);
                    if (o.scalar_type() != t.scalar_type() || o.sizes() != t.sizes() || o.strides() != t.strides())
                        throw "out[" + std::to_string(i) + "] must have the shape, strides and type of tensors[" + std::to_string(i) + "]";
                }
            }
            // what is written gets memory of its own first where it is a lazy clone that still shares its original's; that may move what is read
            for (Py_ssize_t i = 0; i < n; ++i) dst[i] = (int64_t)tensor_at(out, i, "out").mutable_data_ptr();
        }
        for (Py_ssize_t i = 0; i < n; ++i) src[i] = (int64_t)tensor_at(list, i, "tensors").const_data_ptr();
        if (out != Py_None) {
            std::vector<std::pair<int64_t, int64_t>> ranges;       // written memory, and read memory that is not written in place
            ranges.reserve(2 * n);
            for (Py_ssize_t i = 0; i < n; ++i) {
                const int64_t bytes = numel[i] * (types[i] == 0 ? 4 : 2);
                if (bytes == 0) continue;
                ranges.emplace_back(dst[i], bytes);
                if (dst[i] != src[i]) ranges.emplace_back(src[i], -bytes);
            }
            std::sort(ranges.begin(), ranges.end());
            // a written range must not meet any other one; read ranges may meet each other
            int64_t end_written = 0, end_read = 0;
            for (const auto& r : ranges) {
                const bool written = r.second > 0;
                const int64_t end = r.first + (written ? r.second : -r.second);
                if (r.first < end_written || (written && r.first < end_read))
                    throw std::string(out == list ? "the same memory is in the list twice (it would be scaled twice)"
                                                  : "the outputs overlap each other or another gradient");
                int64_t& e = written ? end_written : end_read;
                if (end > e) e = end;
            }
        }
        return Py_BuildValue("(y#N y#y#)", (const char*)src.data(), (Py_ssize_t)(n * 8),
                             out == Py_None ? (Py_INCREF(Py_None), Py_None) : PyBytes_FromStringAndSize((const char*)dst.data(), n * 8),
                             (const char*)numel.data(), (Py_ssize_t)(n * 8), (const char*)types.data(), (Py_ssize_t)(n * 4));
    } catch (const std::string& why) {
        PyErr_SetString(PyExc_ValueError, why.c_str());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_ValueError, "a tensor could not be read");
    }
    return nullptr;
}

static PyMethodDef methods[] = {{"clip_table", clip_table, METH_VARARGS, "addresses, sizes and types of a list of gradient tensors, checked"},
                                {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "vitk_host", nullptr, -1, methods};
PyMODINIT_FUNC PyInit_vitk_host(void) { return PyModule_Create(&module); }
