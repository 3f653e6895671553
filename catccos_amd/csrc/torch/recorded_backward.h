// A backward pass that is recorded into a graph must not add to a leaf whose gradient is accumulated on the default stream: torch would have that stream, which cannot be part of a capture, wait
// for the recording one, and the process ends.  It is so where an eager graph of the leaf, whose node for it is shared, is still alive.
#pragma once
#include <c10/core/Stream.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>

// Whether the node whose backward runs hands a gradient to such a leaf.
inline bool AccumulatesOnDefaultStream()
{
    const auto node = torch::autograd::get_current_node();
    if (!node) return false;
    for (const torch::autograd::Edge &e : node->next_edges()) {
        if (!dynamic_cast<torch::autograd::AccumulateGrad *>(e.function.get())) continue;
        const std::optional<c10::Stream> s = e.function->stream();
        if (s && s->id() == 0) return true;
    }
    return false;
}
