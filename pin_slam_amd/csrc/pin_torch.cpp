// pin_torch.cpp -- what is asked of torch's own objects, many at a time, in a library of its own
// (libpin_slam_torch.so): the kernels' library knows no torch.
//
// An optimiser step needs two addresses and ten properties per parameter.  Asked from Python they
// cost 0.43 us per parameter, which for a few hundred small ones is more than the step's kernels
// (331 parameters, 13M elements: 77 us); here 0.01.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
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

// The gradient of label_log_probs as a node of torch's graph: the engine runs it on a thread of its own, where
// the same in Python takes longer (forward and gradient of 64 x 20 f32: 90 us, here 60; of 16384 x 1003 f16: 105, here 73).
// Outputs log_prob, entropy and, with k > 0, top_log_prob; one input, the logits [n, C].
typedef decltype(&pin_label_logprob_bwd) LabelBwd;

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
        at::Tensor z = logits.unpack(), y = labels.unpack(), idx = k > 0 ? top.unpack() : at::Tensor();
        at::Tensor dz;
        {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard device(z.device());
            if (z.size(1) > 1 && z.stride(1) != 1) z = z.contiguous();   // (kept elsewhere in between)
            y = y.contiguous();
            at::Tensor u[3];
            for (size_t i = 0; i < grads.size() && i < 3; ++i)
                if (grads[i].defined()) u[i] = grads[i].to(at::kFloat).contiguous();
            if (k > 0) idx = idx.contiguous();
            dz = at::empty({z.size(0), z.size(1)}, z.options());
            const auto at_f32 = [](const at::Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; };
            const int type = z.scalar_type() == c10::kFloat  ? PIN_TYPE_F32
                             : z.scalar_type() == c10::kHalf ? PIN_TYPE_F16
                                                             : PIN_TYPE_BF16;
            const int rc = bwd(z.const_data_ptr(), type, z.size(0), z.size(1), z.stride(0), y.const_data_ptr<int64_t>(), ignore,
                               (int32_t)k, k > 0 ? idx.const_data_ptr<int64_t>() : nullptr, stats.const_data_ptr<float>(),
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

// Makes log_prob, entropy and top_log_prob (None with k = 0) results of logits, with what pin_label_logprob left for
// the gradient.  bwd: pin_label_logprob_bwd.  0, or -1 for what are not tensors or cannot be saved.
int pin_torch_label_attach(void* bwd, PyObject* logits, PyObject* labels, PyObject* stats, PyObject* log_prob,
                           PyObject* entropy, PyObject* top_log_prob, PyObject* top_index, int64_t ignore, int64_t k) {
    for (PyObject* o : {logits, labels, stats, log_prob, entropy})
        if (!THPVariable_Check(o)) return -1;
    if (!bwd || (k > 0 && !(THPVariable_Check(top_log_prob) && THPVariable_Check(top_index)))) return -1;
    try {
        const std::shared_ptr<LabelNode> node(new LabelNode(), torch::autograd::deleteNode);
        const at::Tensor& z = THPVariable_Unpack(logits);
        node->set_next_edges(torch::autograd::collect_next_edges(z));
        node->bwd = (LabelBwd)bwd;
        node->logits = torch::autograd::SavedVariable(z, false);
        node->labels = torch::autograd::SavedVariable(THPVariable_Unpack(labels), false);
        if (k > 0) node->top = torch::autograd::SavedVariable(THPVariable_Unpack(top_index), false);
        node->stats = THPVariable_Unpack(stats);
        node->ignore = ignore;
        node->k = k;
        torch::autograd::set_history(THPVariable_Unpack(log_prob), node);
        torch::autograd::set_history(THPVariable_Unpack(entropy), node);
        if (k > 0) torch::autograd::set_history(THPVariable_Unpack(top_log_prob), node);
        return 0;
    } catch (...) {
        return -1;
    }
}

}  // extern "C"
