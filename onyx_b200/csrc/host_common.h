// Host-side helpers that the library's translation units share (defined in masked_select.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace onyx {

// Records a failed launch for onyx_last_cuda_error and maps it to a return code.
int finish_launch(cudaError_t e);

// ONYX_OPTION_PDL: launches carry the programmatic-stream-serialization attribute.
bool pdl_enabled();

}  // namespace onyx
