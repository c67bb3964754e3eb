// Host side shared by the 8-bit KV cache's entry points: argument checks, the
// kernels' argument structs and the device switch.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "kv_cache.cuh"

namespace rtr {

// Strides of the dense K and V rows, in elements.
struct KvRows {
  int64_t k_token, k_head, v_token, v_head;
};

struct KvGrid {
  int64_t items;  // page items (grid x)
  int per_seq;    // items of a sequence without starts
  int units;      // head x (K, V) units a block loops over
  int splits;     // grid y
};

// The reason why the cache or the batch is refused, or null.
const char* kv_check(const rtr_kv_cache* c, const rtr_kv_batch* b);
KvCache kv_device_cache(const rtr_kv_cache* c);
KvBatch kv_device_batch(const rtr_kv_batch* b);
KvGrid kv_page_grid(int rows, int seqs, bool starts, int page, int kv_heads, int sms);

// The device's SM count, asked for once (a call would spend 0.3 us on it each time).
int kv_sms(int device, cudaError_t& e);

// Allows a kernel `bytes` of dynamic shared memory on `device`, the first time (done: a bit a device).
template <typename F> cudaError_t kv_allow_smem(F* kernel, int bytes, std::atomic<uint64_t>& done, int device) {
  const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Launches a kernel of the cache: programmatic dependent launch (every kernel waits for its
// predecessor before it reads anything, so only the launch itself overlaps; a pass of one token of
// attention 8.2 -> 6.3 us, of one written token 4.2 -> 3.4), and the
// blocks along z as one cluster where `cluster` is above 1.
template <typename... KArgs, typename... Args>
cudaError_t kv_launch(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                      Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_on(PDL_ATTN) ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = cluster;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Makes `device` the thread's current one for a call and puts the former back.
struct KvDevice {
  int former = -1, device, sms = 0;
  cudaError_t error;
  explicit KvDevice(int dev) : device(dev) {
    error = cudaGetDevice(&former);
    if (error == cudaSuccess && former != dev) error = cudaSetDevice(dev);
    if (error == cudaSuccess) sms = kv_sms(dev, error);
  }
  ~KvDevice() {
    if (former >= 0 && former != device) cudaSetDevice(former);
  }
};

}  // namespace rtr
