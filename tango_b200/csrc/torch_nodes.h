// Autograd nodes of the host layer's operators (torch_autograd.cpp, torch_rows8.cpp).
#pragma once
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "torch_ops.h"

namespace tango_host {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Below the autograd and view-tracking layers: forward and backward bodies only produce fresh, non-differentiable tensors.
using Raw = at::AutoDispatchBelowADInplaceOrView;

struct OnceNode : Node {
    virtual variable_list backward(const variable_list &grads) = 0;

    variable_list apply(variable_list &&grads) override {
        variable_list out;
        {
            const c10::AutoGradMode no_grad(false);
            const Raw raw;
            out = backward(grads);
        }
        if (!c10::GradMode::is_enabled()) return out;
        bool differentiable = false;
        for (const Tensor &g : grads) differentiable |= g.defined() && g.requires_grad();
        if (!differentiable) return out;
        // a graph of the gradients was asked for: results that raise when they are differentiated again
        for (Tensor &t : out)
            if (t.defined()) {
                t = t.detach();
                t.set_requires_grad(true);
            }
        return torch::autograd::DelayedError("trying to differentiate twice a function that was marked with "
                                             "@once_differentiable", (int)out.size())(std::move(out));
    }
    bool needs(size_t input) const { return task_should_compute_output(input); }
};

// A node whose operands pass through the saved-tensor hooks and are given back after the backward pass.
struct SavingNode : OnceNode {
    std::vector<SavedVariable> saved;
    bool released = false;
    // call it after set_history; the first `outputs` of them are outputs of the node
    void keep(std::initializer_list<Tensor> tensors, size_t outputs = 0) {
        saved.reserve(tensors.size());
        for (const Tensor &t : tensors) {
            saved.emplace_back(t, outputs > 0);
            if (outputs > 0) --outputs;
        }
    }
    std::vector<Tensor> kept() {
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        std::vector<Tensor> t;
        t.reserve(saved.size());
        for (SavedVariable &s : saved) t.push_back(s.unpack(shared_from_this()));
        return t;
    }
    void release_variables() override {
        for (SavedVariable &s : saved) s.reset_data();
        released = true;
    }
};

// The node of an operation on `inputs`, or null when no gradient is recorded.
template <class N, class... T>
std::shared_ptr<N> make_node(const T &...inputs) {
    if (!torch::autograd::compute_requires_grad(inputs...)) return nullptr;
    auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

}  // namespace tango_host
