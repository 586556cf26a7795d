// What the binding files of the module share: argument checks, per-device state.
#pragma once

#include <torch/extension.h>

#define CHECK_CUDA(x) TORCH_CHECK((x).is_cuda(), #x " must be a CUDA tensor")
#define CHECK_BF16(x) TORCH_CHECK((x).scalar_type() == at::kBFloat16, #x " must be bfloat16")
// every tensor a kernel dereferences must live on the launching tensor's CUDA device (a host pointer faults)
#define CHECK_ON(x, ref)                                                                                         \
  TORCH_CHECK((x).is_cuda() && (x).get_device() == (ref).get_device(), #x " must be on the device of " #ref)
#define CHECK_I32(x) TORCH_CHECK((x).scalar_type() == at::kInt, #x " must be int32")
#define CHECK_I64(x) TORCH_CHECK((x).scalar_type() == at::kLong, #x " must be int64")

namespace ecz {

// Streaming multiprocessors of a device (cached).
int device_sms(int device);

// The per-device status word that kernels set when a bounded wait gives up or an index is out of range.
unsigned* device_status(const at::Device& device);

// bindings_train.cpp: the training operators.
void bind_training(pybind11::module_& m);

}  // namespace ecz
