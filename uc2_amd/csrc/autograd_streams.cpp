// The stream that a leaf's gradient is accumulated on: torch fixes it when the accumulation's node is made -- by whichever operation first used the leaf, or
// by a wrapper that holds the node -- and shows it in C++ only.  A Python module of its own: the kernels' library knows no torch types.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

// its id (0: the device's default stream), or None where no such node is alive or the leaf is on no device with streams
static py::object accumulation_stream(const at::Tensor& leaf) {
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return py::none();
  const auto stream = node->stream();
  if (!stream) return py::none();
  return py::cast(static_cast<long long>(stream->id()));
}

PYBIND11_MODULE(_autograd_streams, m) { m.def("accumulation_stream", &accumulation_stream); }
