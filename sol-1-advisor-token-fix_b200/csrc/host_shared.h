// host_shared.h — host-side state that the library's translation units share: the checked
// device (compute capability, SM count, error word) and the cached TMA descriptor encoder.
// Defined in attn_bwd_b200.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace attn_bwd {

struct HostDevice {
  int index;      // CUDA device ordinal
  int sm_count;
  int* err;       // device address of the error word that attn_bwd_b200_poll_error reads
};

// Checks the current device (once per device) and fills *out; returns an ATTN_BWD_E* code.
int host_device(HostDevice* out);

// Encodes (or finds in the cache) a tiled tensor map; false when the driver refuses it.
bool host_make_map(CUtensorMap* m, CUtensorMapDataType dt, int rank, const void* ptr, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle sw);

}  // namespace attn_bwd
