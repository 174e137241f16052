// pybind11 fast path for the PyTorch eager launch.
//
// Same two functions as the reference's extension (pyptx/_shim/torch_ext.cpp:14-80):
//   load_shim(path)      dlopen the C-ABI library and resolve its raw launch entry
//   launch_kernel(handle, stream, inputs, out_shapes, out_dtypes) -> outputs
// launch_kernel allocates the outputs with torch::empty on the first input's device, builds
// the void*[] of inputs then outputs and makes one call into pb200_launch_raw.  Unlike the
// reference, the error buffer is per call (no shared static buffer), and inputs are checked
// for device / contiguity before the call.
//
// Launcher is the same launch with everything static bound to the kernel object: one call from
// Python checks the inputs against the specs, takes the current stream, allocates and launches.
// A call of ours costs the host about as long as a small kernel runs, so this path decides what a
// chain of small calls costs (measured: 4 to 5.5 us a call against 11.5 with the checks in Python).  It answers
// None for whatever it does not accept, and the caller takes the checking path, which words the errors.
#include <torch/extension.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/Context.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <dlfcn.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

namespace {

using LaunchRawFn = int (*)(int64_t, uint64_t, void**, size_t, char*);
LaunchRawFn g_launch_raw = nullptr;
void* g_lib = nullptr;

void load_shim(const std::string& path) {
    void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_GLOBAL);
    if (!lib) throw std::runtime_error(std::string("pyptx_b200: dlopen failed: ") + dlerror());
    void* sym = dlsym(lib, "pb200_launch_raw");
    if (!sym) throw std::runtime_error("pyptx_b200: pb200_launch_raw not found in " + path);
    g_lib = lib;
    g_launch_raw = reinterpret_cast<LaunchRawFn>(sym);
}

std::vector<torch::Tensor> launch_kernel(int64_t handle, int64_t stream,
                                         const std::vector<torch::Tensor>& inputs,
                                         const std::vector<std::vector<int64_t>>& out_shapes,
                                         const std::vector<int64_t>& out_dtypes) {
    if (!g_launch_raw) throw std::runtime_error("pyptx_b200: load_shim() has not been called");
    if (inputs.empty()) throw std::invalid_argument("pyptx_b200: a kernel call requires at least one input");
    if (out_shapes.size() != out_dtypes.size()) throw std::invalid_argument("pyptx_b200: out_shapes / out_dtypes mismatch");
    const auto device = inputs[0].device();
    if (!device.is_cuda()) throw std::invalid_argument("pyptx_b200: inputs must be CUDA tensors (there is no CPU path)");
    std::vector<void*> ptrs;
    ptrs.reserve(inputs.size() + out_shapes.size());
    for (size_t i = 0; i < inputs.size(); ++i) {
        const auto& t = inputs[i];
        if (t.device() != device) throw std::invalid_argument("pyptx_b200: input " + std::to_string(i) + " is on another device");
        if (!t.is_contiguous()) throw std::invalid_argument("pyptx_b200: input " + std::to_string(i) + " is not contiguous");
        ptrs.push_back(t.data_ptr());
    }
    std::vector<torch::Tensor> outs;
    outs.reserve(out_shapes.size());
    for (size_t i = 0; i < out_shapes.size(); ++i) {
        auto opts = torch::TensorOptions().dtype(static_cast<c10::ScalarType>(out_dtypes[i])).device(device);
        outs.push_back(torch::empty(out_shapes[i], opts));
        ptrs.push_back(outs.back().data_ptr());
    }
    char err[128] = {0};
    int rc;
    {
        pybind11::gil_scoped_release nogil;
        rc = g_launch_raw(handle, static_cast<uint64_t>(stream), ptrs.data(), ptrs.size(), err);
    }
    if (rc != 0)
        throw std::runtime_error("pyptx_b200: pb200_launch_raw failed (code " + std::to_string(rc) + "): " + err);
    return outs;
}

class Launcher {
public:
    Launcher(int64_t handle, std::vector<int64_t> in_dtypes, std::vector<std::vector<int64_t>> in_shapes,
             std::vector<int64_t> out_dtypes, std::vector<std::vector<int64_t>> out_shapes, int64_t scratch_bytes)
        : handle_(handle), out_shapes_(std::move(out_shapes)), in_shapes_(std::move(in_shapes)) {
        for (auto d : in_dtypes) in_dtypes_.push_back(static_cast<c10::ScalarType>(d));
        for (auto d : out_dtypes) out_dtypes_.push_back(static_cast<c10::ScalarType>(d));
        n_results_ = out_shapes_.size();
        if (scratch_bytes > 0) {
            out_shapes_.push_back({scratch_bytes});
            out_dtypes_.push_back(c10::ScalarType::Byte);
        }
    }

    // A new reference to one tensor, a tuple of tensors, or None when the inputs are not exactly what the specs say.
    PyObject* call(PyObject* args) const {
        const size_t n_in = in_shapes_.size();
        if (!g_launch_raw || !PyTuple_CheckExact(args) || (size_t)PyTuple_GET_SIZE(args) != n_in || n_in == 0) return decline();
        constexpr size_t kMaxBuffers = 32;
        void* ptrs[kMaxBuffers];
        if (n_in + out_shapes_.size() > kMaxBuffers) return decline();
        c10::Device device(c10::DeviceType::CPU);
        for (size_t i = 0; i < n_in; ++i) {
            PyObject* obj = PyTuple_GET_ITEM(args, (Py_ssize_t)i);
            if (!THPVariable_CheckExact(obj)) return decline();
            const at::Tensor& t = THPVariable_Unpack(obj);
            if (!t.is_cuda() || t.layout() != c10::Layout::Strided || t.scalar_type() != in_dtypes_[i] ||
                t.sizes() != c10::IntArrayRef(in_shapes_[i]) || !t.is_contiguous())
                return decline();
            if (i == 0) device = t.device();
            else if (t.device() != device) return decline();
            ptrs[i] = t.data_ptr();
        }
        if (c10::cuda::current_device() != device.index()) return decline();
        // Allocations that somebody wants to see or have filled go through the dispatcher: a dispatch mode is active, or
        // torch fills what a kernel may leave unwritten (torch.utils.deterministic.fill_uninitialized_memory).
        if (c10::impl::TorchDispatchModeTLS::any_modes_set() ||
            (at::globalContext().deterministicAlgorithms() && at::globalContext().deterministicFillUninitializedMemory()))
            return decline();
        const uint64_t stream = (uint64_t)(uintptr_t)c10::cuda::getCurrentCUDAStream(device.index()).stream();
        c10::SmallVector<at::Tensor, 4> outs;
        for (size_t i = 0; i < out_shapes_.size(); ++i) {
            // torch's caching allocator on the current stream, without the dispatcher
            outs.push_back(at::Tensor(at::detail::empty_cuda(out_shapes_[i], out_dtypes_[i], device, std::nullopt)));
            ptrs[n_in + i] = outs.back().data_ptr();
        }
        char err[128] = {0};
        int rc;
        {
            pybind11::gil_scoped_release nogil;
            rc = g_launch_raw(handle_, stream, ptrs, n_in + outs.size(), err);
        }
        if (rc != 0)
            throw std::runtime_error("pyptx_b200: pb200_launch_raw failed (code " + std::to_string(rc) + "): " + err);
        if (n_results_ == 1) return THPVariable_Wrap(outs[0]);
        PyObject* res = PyTuple_New((Py_ssize_t)n_results_);
        if (!res) return nullptr;
        for (size_t i = 0; i < n_results_; ++i) PyTuple_SET_ITEM(res, (Py_ssize_t)i, THPVariable_Wrap(outs[i]));
        return res;
    }

private:
    static PyObject* decline() { Py_RETURN_NONE; }

    int64_t handle_;
    size_t n_results_ = 0;
    std::vector<std::vector<int64_t>> out_shapes_, in_shapes_;
    std::vector<c10::ScalarType> in_dtypes_, out_dtypes_;
};

// The launcher as a plain C function of Python (its self is a capsule around the Launcher): no argument
// conversion on the way in.
constexpr const char* kCapsule = "pyptx_b200.Launcher";

PyObject* launcher_call(PyObject* self, PyObject* args) {
    try {
        return static_cast<const Launcher*>(PyCapsule_GetPointer(self, kCapsule))->call(args);
    } catch (const c10::Error&) {
        Py_RETURN_NONE;             // torch refused an input or an allocation, nothing is enqueued: let the checking path say so
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
PyMethodDef launcher_method = {"launch", launcher_call, METH_O,
                               "check, allocate and launch; None when the inputs need the checking path"};

pybind11::object make_launcher(int64_t handle, std::vector<int64_t> in_dtypes, std::vector<std::vector<int64_t>> in_shapes,
                               std::vector<int64_t> out_dtypes, std::vector<std::vector<int64_t>> out_shapes, int64_t scratch_bytes) {
    auto* launcher = new Launcher(handle, std::move(in_dtypes), std::move(in_shapes), std::move(out_dtypes), std::move(out_shapes),
                                  scratch_bytes);
    pybind11::object self = pybind11::reinterpret_steal<pybind11::object>(PyCapsule_New(
        launcher, kCapsule, [](PyObject* c) { delete static_cast<Launcher*>(PyCapsule_GetPointer(c, kCapsule)); }));
    if (!self) { delete launcher; throw pybind11::error_already_set(); }
    return pybind11::reinterpret_steal<pybind11::object>(PyCFunction_New(&launcher_method, self.ptr()));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("load_shim", &load_shim, "dlopen the C-ABI library");
    m.def("launch_kernel", &launch_kernel, "allocate outputs and launch a registered kernel");
    m.def("make_launcher", &make_launcher, "the launch of one kernel object with static shapes, as a function of its inputs' tuple");
}
