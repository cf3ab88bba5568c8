// pin_torch.cpp -- what is done with torch's own objects, host code in a library of its own
// (libpin_slam_torch.so): the kernels' library knows no torch.
//
// pin_torch_gather: an optimiser step needs two addresses and ten properties per parameter.  Asked
// from Python they cost 0.43 us per parameter, which for a few hundred small ones is more than the
// step's kernels (331 parameters, 13M elements: 77 us); here 0.01.
// pin_torch_touched: what was written through an address is marked as modified, as torch's own operators do.
// pin_torch_label: label_log_probs' outputs, launch and node in torch's graph, in one call.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/version.h>

#include "pin_slam_amd.h"

namespace {

bool as_taken(const at::Tensor& t, c10::ScalarType type, int64_t device, int64_t size) {
    return t.defined() && t.layout() == c10::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
           !t.is_neg() && t.scalar_type() == type && (device < 0 ? t.is_cpu() : t.is_cuda() && t.get_device() == device) &&
           t.numel() == size && t.is_contiguous();
}

// A tensor with memory of its own that the kernels may read: no wrapper of a transform, a trace or another program's class.
bool has_memory(const at::Tensor& t) {
    const c10::DispatchKeySet keys = t.key_set();
    return t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() && !keys.has(c10::DispatchKey::Functionalize) &&
           !keys.has(c10::DispatchKey::FuncTorchBatched) && !keys.has(c10::DispatchKey::FuncTorchGradWrapper);
}
bool transformed() { return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode); }

// The gradient of label_log_probs as a node of torch's graph: the engine runs it on a thread of its own, where
// the same in Python takes longer (forward and gradient of 16384 x 1003 f16 105 us, with this node 73).
// Outputs log_prob, entropy and, with k > 0, top_log_prob; one input, the logits [n, C].
typedef decltype(&pin_label_logprob_workspace_bytes) LabelWorkspace;
typedef decltype(&pin_label_logprob) LabelFwd;
typedef decltype(&pin_label_logprob_bwd) LabelBwd;

int type_of(c10::ScalarType t) {
    return t == c10::kFloat ? PIN_TYPE_F32 : t == c10::kHalf ? PIN_TYPE_F16 : t == c10::kBFloat16 ? PIN_TYPE_BF16 : -1;
}

struct LabelNode : torch::autograd::Node {
    LabelBwd bwd = nullptr;
    torch::autograd::SavedVariable logits, labels, top;
    at::Tensor stats;
    int64_t ignore = 0, k = 0;

    std::string name() const override { return "LabelLogProbsBackward"; }

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
        labels.reset_data();
        top.reset_data();
        stats.reset();
    }

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        bool plain = !transformed();
        for (const at::Tensor& g : grads) plain = plain && (!g.defined() || has_memory(g));
        TORCH_CHECK_NOT_IMPLEMENTED(plain, "label_log_probs: batched gradients and torch.func's transforms are not implemented");
        at::Tensor z = logits.unpack(), y = labels.unpack(), idx = k > 0 ? top.unpack() : at::Tensor();
        at::Tensor dz;
        {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard device(z.device());
            if (z.size(1) > 1 && z.stride(1) != 1) z = z.contiguous();   // (kept elsewhere in between)
            y = y.contiguous();
            at::Tensor u[3];
            for (size_t i = 0; i < grads.size() && i < 3; ++i)
                if (grads[i].defined()) u[i] = grads[i].to(at::kFloat).resolve_neg().contiguous();
            if (k > 0) idx = idx.contiguous();
            dz = at::empty({z.size(0), z.size(1)}, z.options());
            const auto at_f32 = [](const at::Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; };
            const int rc = bwd(z.const_data_ptr(), type_of(z.scalar_type()), z.size(0), z.size(1), z.stride(0),
                               y.const_data_ptr<int64_t>(), ignore, (int32_t)k, k > 0 ? idx.const_data_ptr<int64_t>() : nullptr, stats.const_data_ptr<float>(),
                               at_f32(u[0]), at_f32(u[1]), at_f32(u[2]), dz.mutable_data_ptr(),
                               (void*)c10::hip::getCurrentHIPStream(z.device().index()).stream());
            TORCH_CHECK(rc == PIN_OK, "pin_label_logprob_bwd failed: ", rc);
        }
        if (!at::GradMode::is_enabled()) return {dz};
        // the gradient has none of its own: asking for one is an error, not zero
        dz.set_requires_grad(true);
        auto once = std::make_shared<torch::autograd::DelayedError>("label_log_probs: trying to differentiate twice", 1);
        return (*once)({dz});
    }
};

// Another thread may go on in Python meanwhile.
struct NoInterpreter {
    PyThreadState* state = PyEval_SaveThread();
    ~NoInterpreter() { PyEval_RestoreThread(state); }
};

// What allocates and launches a forward pass: 14.5 us a call from Python, here 8.7 (1 x 32768 bf16, whose kernel takes 8.0).
void label_forward(LabelWorkspace workspace, LabelFwd forward, LabelBwd backward, const at::Tensor& z, const at::Tensor& y,
                   int64_t k, int64_t ignore, bool grad, at::Tensor& lp, at::Tensor& ent, at::Tensor& top_lp,
                   at::Tensor& top_idx) {
    TORCH_CHECK_NOT_IMPLEMENTED(has_memory(z) && has_memory(y) && !transformed(),
                                "label_log_probs: torch.func's transforms and tensors without memory are not implemented");
    TORCH_CHECK_NOT_IMPLEMENTED(!z._fw_grad(0).defined(), "label_log_probs: forward-mode differentiation is not implemented");
    const int64_t n = z.size(0), c = z.size(1);
    const c10::DeviceGuard device(z.device());
    const at::TensorOptions f32 = at::TensorOptions(z.device()).dtype(at::kFloat);
    at::Tensor stats, ws;
    lp = at::empty({n}, f32);
    ent = at::empty({n}, f32);
    top_lp = at::empty({n, k}, f32);
    top_idx = at::empty({n, k}, f32.dtype(at::kLong));
    if (grad) stats = at::empty({n, 3}, f32);
    const int type = type_of(z.scalar_type());
    const int64_t need = workspace(n, c, type, (int32_t)k);
    if (need > 0) ws = at::empty({need}, f32.dtype(at::kByte));
    const int rc = forward(z.const_data_ptr(), type, n, c, z.stride(0), y.const_data_ptr<int64_t>(), ignore, (int32_t)k,
                           lp.mutable_data_ptr<float>(), ent.mutable_data_ptr<float>(),
                           grad ? stats.mutable_data_ptr<float>() : nullptr, k > 0 ? top_lp.mutable_data_ptr<float>() : nullptr,
                           k > 0 ? top_idx.mutable_data_ptr<int64_t>() : nullptr, need > 0 ? ws.mutable_data_ptr() : nullptr,
                           (void*)c10::hip::getCurrentHIPStream(z.device().index()).stream());
    TORCH_CHECK(rc == PIN_OK, "pin_label_logprob failed: ", rc);
    if (!grad) return;
    const std::shared_ptr<LabelNode> node(new LabelNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(z));
    node->bwd = backward;
    node->logits = torch::autograd::SavedVariable(z, false);
    node->labels = torch::autograd::SavedVariable(y, false);
    if (k > 0) node->top = torch::autograd::SavedVariable(top_idx, false);
    node->stats = stats;
    node->ignore = ignore;
    node->k = k;
    torch::autograd::set_history(lp, node);
    torch::autograd::set_history(ent, node);
    if (k > 0) torch::autograd::set_history(top_lp, node);
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
        return type_of(type);
    } catch (...) {
        return -1;
    }
}

// tensors: a list of tensors that a kernel writes through their addresses.  Their versions are raised, on which
// torch's check of saved tensors and this package's derived views go (tensors made in inference mode have none).
// 0, or -1 where one of them is no tensor.  Called with the interpreter's lock; no exception leaves it.
int pin_torch_touched(PyObject* tensors) {
    if (!PyList_CheckExact(tensors)) return -1;
    try {
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(tensors); ++i) {
            PyObject* o = PyList_GET_ITEM(tensors, i);
            if (!THPVariable_Check(o)) return -1;
            const at::Tensor& t = THPVariable_Unpack(o);
            if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
        return 0;
    } catch (...) {
        return -1;
    }
}

// label_log_probs of checked arguments: logits [n, C] with adjacent classes, labels [n] int64 without gaps, on one device;
// workspace, forward, backward: the kernels' library's entry points.  A new tuple (log_prob, entropy, top_log_prob,
// top_index), results of logits where grad is set; an exception of Python's where that cannot be.
PyObject* pin_torch_label(void* workspace, void* forward, void* backward, PyObject* logits, PyObject* labels, int64_t k,
                          int64_t ignore, int32_t grad) {
    if (!workspace || !forward || !backward || !THPVariable_Check(logits) || !THPVariable_Check(labels)) {
        PyErr_SetString(PyExc_TypeError, "label_log_probs: two tensors");
        return nullptr;
    }
    HANDLE_TH_ERRORS
    const at::Tensor &z = THPVariable_Unpack(logits), &y = THPVariable_Unpack(labels);
    at::Tensor lp, ent, top_lp, top_idx;
    {
        const NoInterpreter released;
        label_forward((LabelWorkspace)workspace, (LabelFwd)forward, (LabelBwd)backward, z, y, k, ignore, grad != 0, lp, ent,
                      top_lp, top_idx);
    }
    PyObject* out = PyTuple_New(4);
    if (!out) return nullptr;
    int at = 0;
    for (const at::Tensor* t : {&lp, &ent, &top_lp, &top_idx}) PyTuple_SET_ITEM(out, at++, THPVariable_Wrap(*t));
    return out;
    END_HANDLE_TH_ERRORS
}

}  // extern "C"
