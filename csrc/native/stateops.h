#pragma once
#include <stdint.h>

#include "../hip/tpi_hip.h"  // plain C structs shared with the device path

namespace tpi {

// Host implementations of csrc/hip/dropout.hip and csrc/hip/pages.hip, bit for bit; addresses
// in the arguments are host memory.  The pages' functions give the reason of a refusal in the
// pool's header, as the kernels do.
void dropout(const tpi_dropout_args& a, int threads);
void pages_copy(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n);
void pages_fork(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n);
void pages_extend(const tpi_pages& p, const int64_t* slots, const int64_t* more, int64_t n);
void pages_free(const tpi_pages& p, const int64_t* slots, int64_t n);
void pages_compact(const tpi_pages& p, bool clear);

}  // namespace tpi
