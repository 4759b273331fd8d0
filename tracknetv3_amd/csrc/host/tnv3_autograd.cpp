// tnv3_autograd.cpp -- libtnv3_autograd.so: what a layer's backward pass has to know about autograd's graph and torch's Python API does not tell.
// Host code against torch's own headers; tracknetv3_amd/_lib.py binds it (ctypes, with the interpreter's lock held).
#include <Python.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_function.h>

// ctx: a torch.autograd.Function's context inside its backward.  The most of `capacity` stream ids that fit, of the nodes that take the gradients which
// the running pass wants (a node runs on the stream that was current when it was made; 0 is the default stream, -1 stands for no stream: CPU); returns how
// many there are, -1 if the graph is gone.
extern "C" int tnv3_gradient_streams(PyObject* ctx, long long* streams, int capacity) {
  try {
    const auto node = reinterpret_cast<THPFunction*>(ctx)->cdata.lock();
    if (!node) return -1;
    int count = 0;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
      const auto& next = node->next_edge(i).function;
      if (!next || !node->task_should_compute_output(i)) continue;
      const auto stream = next->stream();
      if (count < capacity) streams[count] = stream ? static_cast<long long>(stream->id()) : -1;
      ++count;
    }
    return count;
  } catch (...) {
    return -1;
  }
}
