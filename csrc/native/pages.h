#pragma once
#include <stdint.h>

#include "../hip/tpi_hip.h"  // plain C structs shared with the device path

namespace tpi {

// Host implementations of csrc/hip/pages.hip; addresses in `p` are host memory.  The reason of a
// refusal goes to the pool's header, as the kernels do it.
void pages_copy(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n);
void pages_fork(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n);
void pages_extend(const tpi_pages& p, const int64_t* slots, const int64_t* more, int64_t n);
void pages_free(const tpi_pages& p, const int64_t* slots, int64_t n);
void pages_compact(const tpi_pages& p, bool clear);

}  // namespace tpi
