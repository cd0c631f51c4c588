// Tensor allocation with the GIL released (Checkpointer.materialize).
//
// A successor that materializes its state group by group allocates on a background thread
// while its main thread restores the groups already allocated.  An allocation of HBM that its
// predecessor has only just freed blocks inside the driver until the memory is cleared --
// measured on MI355X, up to 15 s behind a 170 GB spill -- and torch.empty() holds the GIL
// all that time, so the restoring thread could not even return from its (GIL-free) engine
// call.  at::empty here is the same caching-allocator allocation, without the GIL.
#include <torch/extension.h>

#include <vector>

#include "torchext.h"

namespace {

at::Tensor empty_nogil(const std::vector<int64_t>& shape, const at::Tensor& like) {
  const at::TensorOptions options = like.options();
  py::gil_scoped_release nogil;
  return at::empty(shape, options);
}

}  // namespace

namespace tpi {

uint64_t (*hip_stream_of)(int device);  // set by hip_stream.cpp

static HipApi g_hip;

const HipApi& hip_api() {
  if (!g_hip.dropout) throw HipFailure("libtpi_hip.so is not loaded");
  return g_hip;
}

void hip_check(int rc, const char* what) {
  if (rc != 0) throw HipFailure(std::string(what) + " failed: " + hip_api().last_error());
}

}  // namespace tpi

PYBIND11_MODULE(_tpi_torch, m) {
  m.doc() = "torch helpers that release the GIL, torch operators and their launches "
            "(terraform_provider_iterative_amd)";
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const tpi::HipFailure& e) {
      const auto type =
          py::module_::import("terraform_provider_iterative_amd.ops._loader").attr("HipError");
      PyErr_SetString(type.ptr(), e.what());
    }
  });
  m.def("use_hip", [](const std::vector<uintptr_t>& at) {
    if (at.size() != 8) throw std::invalid_argument("use_hip: addresses of 8 entry points");
    tpi::g_hip = {(decltype(&tpi_last_error))at[0],  (decltype(&tpi_dropout))at[1],
                  (decltype(&tpi_pages_copy))at[2],  (decltype(&tpi_pages_fork))at[3],
                  (decltype(&tpi_pages_extend))at[4], (decltype(&tpi_pages_free))at[5],
                  (decltype(&tpi_pages_compact))at[6], (decltype(&tpi_capture_id))at[7]};
  });
  m.def("stream_and_capture", [](int device) {
    const uint64_t stream = tpi::current_stream(device);
    uint64_t capture = 0;
    tpi::hip_check(tpi::hip_api().capture_id(stream, &capture), "capture_id");
    return std::make_pair(stream, capture);
  }, "current stream of a device, and the number of the capture that it is part of (0: none)");
  tpi::bind_dropout(m);
  tpi::bind_pages(m);
  m.def("empty", &empty_nogil, "at::empty(shape, like.options()) with the GIL released",
        py::arg("shape"), py::arg("like"));
}
