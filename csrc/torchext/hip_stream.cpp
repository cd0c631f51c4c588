// torch's current stream of a device: the one part of _tpi_torch that needs a torch built for ROCm
// (_build.py leaves it out for any other).
#include <c10/hip/HIPStream.h>

#include "streams.h"

namespace tpi {

static uint64_t stream_of(int device) {
  return (uint64_t)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
}

static const bool g_set = (hip_stream_of = &stream_of, true);

}  // namespace tpi
