// Launches of csrc/hip/pages.hip on the current stream of a pool's device (ops/paging.py); the
// pool's description is the bytes of a tpi_pages.  Each returns the stream.
#include <string.h>

#include "torchext.h"

namespace tpi {

namespace {

struct Pool {
  tpi_pages p;
  c10::DeviceGuard guard;
  uint64_t stream;
  Pool(const py::bytes& raw, int device) : guard(c10::Device(c10::kCUDA, device)) {
    const std::string_view bytes = raw;
    if (bytes.size() != sizeof(tpi_pages)) throw std::invalid_argument("not a pool's description");
    memcpy(&p, bytes.data(), sizeof(p));
    stream = current_stream(device);
  }
};

const void* address(uintptr_t a) { return (const void*)a; }

}  // namespace

void bind_pages(py::module_& m) {
  m.def("pages_copy", [](const py::bytes& raw, int device, uintptr_t src, uintptr_t dst,
                         int64_t n, int wide) {
    const Pool pool(raw, device);
    hip_check(hip_api().pages_copy(&pool.p, address(src), address(dst), n, wide, pool.stream),
              "copy");
    return pool.stream;
  });
  m.def("pages_fork", [](const py::bytes& raw, int device, uintptr_t src, uintptr_t dst,
                         int64_t n, int wide) {
    const Pool pool(raw, device);
    hip_check(hip_api().pages_fork(&pool.p, address(src), address(dst), n, wide, pool.stream),
              "fork");
    return pool.stream;
  });
  m.def("pages_extend", [](const py::bytes& raw, int device, uintptr_t slots, int64_t n, int wide,
                           uintptr_t more, int64_t each) {
    const Pool pool(raw, device);
    hip_check(hip_api().pages_extend(&pool.p, address(slots), n, wide, address(more), each,
                                     pool.stream),
              "extend");
    return pool.stream;
  });
  m.def("pages_free", [](const py::bytes& raw, int device, uintptr_t slots, int64_t n, int wide) {
    const Pool pool(raw, device);
    hip_check(hip_api().pages_free(&pool.p, address(slots), n, wide, pool.stream), "free");
    return pool.stream;
  });
  m.def("pages_compact", [](const py::bytes& raw, int device, int clear) {
    const Pool pool(raw, device);
    hip_check(hip_api().pages_compact(&pool.p, clear, pool.stream), "compact");
    return pool.stream;
  });
}

}  // namespace tpi
