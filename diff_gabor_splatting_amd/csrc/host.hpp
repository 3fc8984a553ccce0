// What the C++ host functions share: the entry point table's reader, checks,
// and tensors as the C ABI takes them.
#pragma once

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

namespace gs_host {

namespace py = pybind11;

template <typename F>
void take(const py::dict& table, const char* name, F& slot) {
  if (!table.contains(name))
    throw std::runtime_error(std::string("the entry point table lacks ") + name);
  const auto address = table[name].cast<uintptr_t>();
  if (address == 0) throw std::runtime_error(std::string("null address for ") + name);
  slot = reinterpret_cast<F>(address);
}

[[noreturn]] inline void fail(const std::string& message) { throw std::runtime_error(message); }

inline void require(bool ok, const char* message) {
  if (!ok) fail(message);
}

inline void* stream_of(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

template <typename T>
inline T* ptr(const at::Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

template <typename T>
inline T* ptr(const std::optional<at::Tensor>& t) {
  return t ? ptr<T>(*t) : nullptr;
}

inline at::TensorOptions on(const at::Device& device, at::ScalarType type) {
  return at::TensorOptions().dtype(type).device(device);
}

inline at::Tensor workspace(size_t bytes, const at::Device& device) {
  return at::empty({std::max<int64_t>(int64_t(bytes), 1)}, on(device, at::kByte));
}

// The decoder layers' host functions (layers_host.cpp).
void bind_layers(const py::dict& table);
std::vector<std::string> layer_entry_points();
void define_layers(py::module_& m);

}  // namespace gs_host
