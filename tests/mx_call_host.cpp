// lich_b200/csrc/mx_call.cpp as it stands, for tests without a GPU: CPU tensors pass for tensors of device 0, every thread
// has a stream of its own, and a thread that has given up the interpreter lock is held for a moment, so that whatever it
// still reads of what threads share can be replaced meanwhile.
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pthread.h>
#include <unistd.h>

#include <cstdint>
#include <cstring>
#include <new>
#include <stdexcept>
#include <vector>

namespace c10::cuda {
struct HostStream {
  cudaStream_t stream() const { return reinterpret_cast<cudaStream_t>(pthread_self()); }
};
inline HostStream host_stream(c10::DeviceIndex) { return {}; }
inline c10::DeviceIndex host_device() { return 0; }
}  // namespace c10::cuda

namespace {
PyThreadState* save_and_wait() {
  PyThreadState* s = PyEval_SaveThread();
  usleep(3000);
  return s;
}
}  // namespace

#define is_cuda() is_cpu()
#define get_device() is_cpu() - 1
#define current_device() host_device()
#define getCurrentCUDAStream host_stream
#define PyEval_SaveThread save_and_wait

#include "../lich_b200/csrc/mx_call.cpp"
