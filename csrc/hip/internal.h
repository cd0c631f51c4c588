// Internals shared by the translation units of libtpi_hip.so (not part of the C ABI).
#pragma once
#include <hip/hip_runtime.h>

#include <string>
#include <tuple>

// Sets the thread's tpi_last_error() text; returns -1.
int tpi_fail(const std::string& what);

// Launches a kernel and returns that launch's own error.  hipGetLastError() behind <<<>>> also returns
// what some earlier call of this thread has left there, after its caller has dealt with it: work
// that has begun would be reported as failed, and of several launches the rest left out.
template <typename... P, typename... A>
static inline hipError_t tpi_launch(void (*kernel)(P...), dim3 grid, uint32_t block,
                                    hipStream_t stream, A... a) {
  std::tuple<P...> args(a...);
  return std::apply(
      [&](P&... each) {
        void* list[] = {(void*)&each...};
        return hipLaunchKernel((const void*)kernel, grid, dim3(block), list, 0, stream);
      },
      args);
}

// Sets tpi_last_error() to a failed call's; returns -1.  The runtime remembers the error too, and a later
// look at hipGetLastError() (torch's, behind its own kernels) would take it for its own: it is
// reported here, and taken back there.
static inline int tpi_hip_fail(const char* what, hipError_t error) {
  (void)hipGetLastError();
  return tpi_fail(std::string(what) + ": " + hipGetErrorString(error));
}

#define TPI_HIP(expr)                                       \
  do {                                                      \
    hipError_t e_ = (expr);                                 \
    if (e_ != hipSuccess) return tpi_hip_fail(#expr, e_);   \
  } while (0)

// SDMA device -> host copies (sdma.cpp).  tpi_sdma_open returns nullptr when the lanes are
// off (TPI_D2H_ENGINE=blit, no HSA runtime to bind, no engine): callers then use
// hipMemcpyAsync.  A lane is one completion signal; a pipeline gives each staging buffer its
// own lane and waits on it (host side) before the buffer is written again.
struct tpi_sdma;
tpi_sdma* tpi_sdma_open(int device, int lanes);
void tpi_sdma_close(tpi_sdma* s);
uint32_t tpi_sdma_engine(const tpi_sdma* s);
int tpi_sdma_d2h(tpi_sdma* s, int lane, void* host_dst, const void* dev_src, size_t n);
// Host -> device lanes on an engine off HIP's own H2D engine and the saves' D2H engine
// (TPI_H2D_ENGINE=sdma<i> pins one); nullptr when none is free.
tpi_sdma* tpi_sdma_open_h2d(int device, int lanes);
int tpi_sdma_h2d(tpi_sdma* s, int lane, void* dev_dst, const void* host_src, size_t n);
int tpi_sdma_wait(tpi_sdma* s, int lane);
int tpi_sdma_wait_all(tpi_sdma* s);
