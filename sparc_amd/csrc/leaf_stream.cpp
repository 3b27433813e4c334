// The stream of a leaf's node in torch's autograd graph, which Python cannot see.
//
// The node that accumulates into leaf.grad is made by the first operation on the leaf that records a gradient, keeps the
// stream that was current then, and lives as long as any graph that it is in.  A backward that is captured while a node made
// on the default stream lives would let that stream, which cannot be captured, wait for the capture.
//     sparc_amd::leaf_stream(Tensor leaf) -> int     the stream's number, 0 for the default stream, -1 where no node lives
#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

namespace {

int64_t leaf_stream(const at::Tensor& leaf) {
    if (!leaf.is_leaf()) return -1;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!node) return -1;
    const auto stream = node->stream();
    return stream ? stream->id() : -1;
}

}  // namespace

TORCH_LIBRARY(sparc_amd, m) { m.def("leaf_stream(Tensor leaf) -> int", &leaf_stream); }
