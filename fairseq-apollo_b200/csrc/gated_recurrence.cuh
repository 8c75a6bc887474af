// Interface of the gated linear recurrence (gated_recurrence.cu) to the other translation units.
#pragma once
#include <cuda_runtime.h>

namespace mega {

cudaError_t gated_recurrence_read_device_error(int* v, bool reset);

}  // namespace mega
