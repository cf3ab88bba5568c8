// pin_torch.cpp -- what is asked of torch's own objects, many at a time, in a library of its own
// (libpin_slam_torch.so): the kernels' library knows no torch.
//
// An optimiser step needs two addresses and ten properties per parameter.  Asked from Python they
// cost 0.43 us per parameter, which for a few hundred small ones is more than the step's kernels
// (331 parameters, 13M elements: 77 us); here 0.01.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "pin_slam_amd.h"

namespace {

bool as_taken(const at::Tensor& t, c10::ScalarType type, int64_t device, int64_t size) {
    return t.defined() && t.layout() == c10::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
           !t.is_neg() && t.scalar_type() == type && (device < 0 ? t.is_cpu() : t.is_cuda() && t.get_device() == device) &&
           t.numel() == size && t.is_contiguous();
}

}  // namespace

extern "C" {

// the version that this was built for
const char* pin_torch_version() { return TORCH_VERSION; }

// params: a list of `count` tensors.  Where all of them and their gradients are plain, of one type, contiguous, on
// `device` (-1: the host) and of these sizes: their addresses, and the type (PIN_TYPE_*).  Otherwise -1.
// Called with the interpreter's lock; no exception leaves it.
int pin_torch_gather(PyObject* params, int64_t count, const int64_t* sizes, int64_t device, uint64_t* ps, uint64_t* gs) {
    if (!PyList_CheckExact(params) || PyList_GET_SIZE(params) != count || count < 1) return -1;
    try {
        c10::ScalarType type = c10::ScalarType::Undefined;
        for (int64_t i = 0; i < count; ++i) {
            PyObject* o = PyList_GET_ITEM(params, i);
            if (!THPVariable_CheckExact(o)) return -1;
            const at::Tensor& p = THPVariable_Unpack(o);
            if (!p.defined() || !p.is_leaf()) return -1;
            if (i == 0) type = p.scalar_type();
            const at::Tensor& g = p.grad();
            if (!as_taken(p, type, device, sizes[i]) || !as_taken(g, type, device, sizes[i])) return -1;
            ps[i] = (uint64_t)(uintptr_t)p.mutable_data_ptr();
            gs[i] = (uint64_t)(uintptr_t)g.const_data_ptr();
        }
        return type == c10::kFloat ? PIN_TYPE_F32 : type == c10::kHalf ? PIN_TYPE_F16 : type == c10::kBFloat16 ? PIN_TYPE_BF16 : -1;
    } catch (...) {
        return -1;
    }
}

}  // extern "C"
