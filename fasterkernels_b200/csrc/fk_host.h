// fk_host.h -- host-side helpers shared by the translation units of the
// library: the error string, programmatic dependent launch, the device a call
// runs on.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace fk {

int fail(int code, const char* fmt, ...);  // sets fk_last_error(), returns code
bool pdl_enabled();                        // FK_DECODE_PDL
int pointer_device(const void* p, const char* name, int* device);  // the device `p` lives on

// Makes `device` current for a scope.
struct DeviceScope {
  int prev = 0, dev;
  explicit DeviceScope(int device) : dev(device) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceScope() {
    if (prev != dev) cudaSetDevice(prev);
  }
};

// Launches a kernel that begins with griddepcontrol.wait, so that its blocks
// may be scheduled while the kernel before it in the stream drains.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace fk
