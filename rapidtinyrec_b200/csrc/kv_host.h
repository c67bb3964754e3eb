// Host side shared by the 8-bit KV cache's entry points: argument checks, the
// kernels' argument structs and the device switch.
#pragma once

#include <cuda_runtime.h>

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

// Makes `device` the thread's current one for a call and puts the former back.
struct KvDevice {
  int former = -1, device, sms = 0;
  cudaError_t error;
  explicit KvDevice(int dev) : device(dev) {
    error = cudaGetDevice(&former);
    if (error == cudaSuccess && former != dev) error = cudaSetDevice(dev);
    if (error == cudaSuccess) error = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  ~KvDevice() {
    if (former >= 0 && former != device) cudaSetDevice(former);
  }
};

}  // namespace rtr
