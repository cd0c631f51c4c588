// Streams of a device, for the translation units of _tpi_torch.
#pragma once
#include <stdint.h>

namespace tpi {

// torch's current stream of a device, as HIP's handle; null in a build without hip_stream.cpp.
extern uint64_t (*hip_stream_of)(int device);

}  // namespace tpi
