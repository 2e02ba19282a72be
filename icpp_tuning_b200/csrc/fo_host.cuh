// fo_host.cuh -- host helpers of the C ABI shared by its translation units (defined in
// fo_api.cu): the calling thread's error message, the current device, tensor maps and the
// launch counter.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace fo {

// Queries and attributes enqueue nothing, but a global-mode stream capture on another
// thread would refuse them: this thread runs them in relaxed mode.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

struct HostDevice {
  int dev;
  int sms;
  int* status;  // device status word (record_error)
  unsigned long long timeout_ns;
};

// Sets the calling thread's message and returns `code`.
int host_fail(int code, const char* fmt, ...);
int host_ok();
// FO_OK and the current device, or FO_ENODEVICE / FO_ECUDA with the message set.
int host_device(HostDevice* out);
// 2-D row-major map [outer, inner] with 128-byte swizzled boxes of box_inner x box_outer.
int host_tmap(CUtensorMap* m, int dt, const void* base, uint64_t inner, uint64_t outer, uint64_t row_bytes,
              uint32_t box_inner, uint32_t box_outer, const char* what);
// fp32 planes [planes, outer, inner], rows `row_bytes` apart, boxes of 32 x 32 x 1.
int host_tmap_planes(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint64_t planes, uint64_t row_bytes,
                     const char* what);
void host_count_launches(int n);

inline bool host_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launches `kern` as a programmatic dependent of the previous kernel on the stream (the
// kernel calls griddep_wait before its first global access), as clusters of `cluster` CTAs
// along x when cluster > 1.  More than the default 48 KB of shared memory (static and
// dynamic) is opted in once per device and kernel.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kern)(Params...), std::atomic<uint64_t>& opted, dim3 grid, dim3 block, int smem, int cluster,
                       cudaStream_t stream, Args... args) {
  if (smem > 32 * 1024) {
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if ((opted.load(std::memory_order_acquire) & bit) == 0) {
      RelaxedCapture relaxed;
      cudaFuncAttributes fa;  // the block's 227 KB hold its static shared memory too
      cudaError_t e = cudaFuncGetAttributes(&fa, kern);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448 - static_cast<int>(fa.sharedSizeBytes));
      if (e != cudaSuccess) return e;
      opted.fetch_or(bit, std::memory_order_acq_rel);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace fo
