// What the translation units of the library share on the host: the per-device state that b200fp8_api.cu keeps.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace b200fp8 {

struct HostDevice {
    int sm_count;
    int* status;      // DEVICE status word of b200fp8_device_status
    CUresult (*encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                       const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                       CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    bool pdl;         // launch with programmatic stream serialization
    int debug;        // 512: a kernel leaves one block of its ring unloaded (exercises the bounded waits)
};

// state of the current device, made on its first use
cudaError_t host_device(HostDevice* out);
// one more kernel launched by this thread (b200fp8_launch_count)
void count_launch();

}  // namespace b200fp8
