// Where the nodes of an autograd graph were made: torch runs a node's backward on the stream that was current when the node was
// made, and tells Python nothing of that stream.  Host code only; a library of its own (libcvn_autograd.so), since it is bound to
// torch's C++ interface.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <c10/core/impl/VirtualGuardImpl.h>

#include <memory>
#include <set>
#include <unordered_set>
#include <utility>
#include <vector>

// The streams but the current one of their device that the nodes which this tensor's gradient reaches were made on, each once: their
// number, the first `most` of them in ids and devices; -1 on an exception.  A leaf that no graph holds has no node yet.  A leaf's
// node on no stream (on the CPU) counts as stream 0 of device -1.
extern "C" __attribute__((visibility("default"))) int cvn_graph_streams(PyObject* tensor, int64_t* ids, int* devices, int most) {
  try {
    if (!THPVariable_Check(tensor)) return -1;
    const at::Tensor& t = THPVariable_Unpack(tensor);
    std::shared_ptr<torch::autograd::Node> first = t.grad_fn();
    if (!first) first = torch::autograd::impl::try_get_grad_accumulator(t);
    std::vector<torch::autograd::Node*> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    std::set<std::pair<int, int64_t>> found;
    if (first) todo.push_back(first.get()), seen.insert(first.get());
    while (!todo.empty()) {
      torch::autograd::Node* const node = todo.back();
      todo.pop_back();
      const auto stream = node->stream();
      if (stream) {
        if (*stream != c10::impl::VirtualGuardImpl(stream->device_type()).getStream(stream->device()))
          found.emplace(stream->device_index(), stream->id());
      } else if (node->num_outputs() == 0) {
        found.emplace(-1, 0);
      }
      for (const auto& edge : node->next_edges())
        if (edge.function && seen.insert(edge.function.get()).second) todo.push_back(edge.function.get());
    }
    int n = 0;
    for (const auto& f : found) {
      if (n < most) devices[n] = f.first, ids[n] = f.second;
      ++n;
    }
    return n;
  } catch (...) {
    return -1;
  }
}
