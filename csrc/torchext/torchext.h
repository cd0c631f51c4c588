// Shared by the translation units of _tpi_torch.
#pragma once
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "../hip/tpi_hip.h"
#include "streams.h"

namespace tpi {

// Entry points of libtpi_hip.so, handed over by Python once it has loaded the library (this
// module does not link it: CPU ranks never load it).
struct HipApi {
  decltype(&tpi_last_error) last_error;
  decltype(&tpi_dropout) dropout;
  decltype(&tpi_pages_copy) pages_copy;
  decltype(&tpi_pages_fork) pages_fork;
  decltype(&tpi_pages_extend) pages_extend;
  decltype(&tpi_pages_free) pages_free;
  decltype(&tpi_pages_compact) pages_compact;
  decltype(&tpi_capture_id) capture_id;
};
const HipApi& hip_api();  // throws when the library has not been handed over

// A failed call, raised in Python as ops.HipError.
struct HipFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void hip_check(int rc, const char* what);

inline uint64_t current_stream(c10::DeviceIndex device) {
  if (!hip_stream_of) throw HipFailure("this torch is not built for ROCm");
  return hip_stream_of(device);
}

void bind_dropout(py::module_& m);
void bind_pages(py::module_& m);

}  // namespace tpi
