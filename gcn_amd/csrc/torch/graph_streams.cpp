// torch.ops.gcn_amd.graph_streams: the streams an autograd graph belongs to.  A backward pass waits for the stream of every
// node it runs; while it is being recorded, a node of a stream that takes no part in the recording ends the capture and the
// process.  Python sees the nodes but not their streams.  Built against torch's headers, apart from libgcn_hip.so, which
// knows nothing of torch.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <set>
#include <utility>
#include <vector>

// (device, stream id) of every node below the tensors, each pair once, one after the other.  A leaf's node is the
// accumulator of its gradient, which exists only while something holds it.
static std::vector<int64_t> graph_streams(at::TensorList tensors) {
    std::vector<std::shared_ptr<torch::autograd::Node>> roots;
    std::vector<torch::autograd::Node*> below;
    for (const at::Tensor& t : tensors) {
        if (!t.defined() || !t.requires_grad()) continue;
        auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
        if (!node) continue;
        below.push_back(node.get());
        roots.push_back(std::move(node));
    }
    std::set<torch::autograd::Node*> seen;
    std::set<std::pair<int64_t, int64_t>> streams;
    while (!below.empty()) {
        torch::autograd::Node* node = below.back();
        below.pop_back();
        if (!seen.insert(node).second) continue;
        if (const auto stream = node->stream()) streams.emplace(stream->device_index(), stream->id());
        for (const auto& edge : node->next_edges())
            if (edge.function) below.push_back(edge.function.get());
    }
    std::vector<int64_t> out;
    for (const auto& [device, id] : streams) {
        out.push_back(device);
        out.push_back(id);
    }
    return out;
}

TORCH_LIBRARY(gcn_amd, m) { m.def("graph_streams(Tensor[] tensors) -> int[]", graph_streams); }
