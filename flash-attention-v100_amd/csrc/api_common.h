// What the files of the PyTorch extension share.
#ifndef API_COMMON_H_
#define API_COMMON_H_

#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstring>

namespace api {

inline void check_arch(int device) {
  // The property query copies a structure of more than a kilobyte; the answer never changes.
  static std::atomic<bool> known_gfx950[64];
  if (device >= 0 && device < 64 && known_gfx950[device].load(std::memory_order_relaxed)) return;
  hipDeviceProp_t prop;
  TORCH_CHECK(hipGetDeviceProperties(&prop, device) == hipSuccess, "hipGetDeviceProperties failed");
  TORCH_CHECK(std::strncmp(prop.gcnArchName, "gfx950", 6) == 0, "This repo only supports gfx950 (MI355X) GPUs, got ",
              prop.gcnArchName);
  if (device >= 0 && device < 64) known_gfx950[device].store(true, std::memory_order_relaxed);
}

// torch.empty without the dispatcher, which costs more than the allocation itself.
inline at::Tensor gpu_empty(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, dtype, like.device(), std::nullopt));
}

// Makes the device of a tensor the current one, which it nearly always is: asking is cheaper than setting it and back.
struct OnDeviceOf {
  c10::OptionalDeviceGuard guard;
  explicit OnDeviceOf(const at::Tensor& x) {
    if (c10::hip::current_device() != x.get_device()) guard.reset_device(x.device());
  }
};

}  // namespace api
#endif  // API_COMMON_H_
