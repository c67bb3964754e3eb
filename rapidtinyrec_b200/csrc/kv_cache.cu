// 8-bit KV cache: quantising rows into pages (write) and reading them back.
//
// A page's scale is a power of two: the least one, from 2^-48 to 2^48, at which
// the largest magnitude written to the page (of one head, K or V) is at most
// 448, the largest e4m3 value.  A power of two costs no precision, because e4m3
// is a floating type (4 significant bits over 15 octaves): x / scale and
// code * scale are exact, and when a later token needs a larger scale the codes
// that the page holds are rounded again only where they fall below e4m3's normal
// range.  The result of a call is a function of the page and the new rows alone.
//
// Both kernels give a block one page of one sequence and let it loop over heads
// and K / V ("units"): finding the page costs three dependent loads (starts,
// lens, table), which a block per head would repeat.  Threads take 16 bytes of
// the dense side each, consecutive threads consecutive bytes, so the dense rows
// move in whole lines and the codes in runs of 4 (fp32) or 8 (bf16) bytes a
// thread.  Both are bound by HBM once a call has some thousand rows.
#include <cuda_runtime.h>

#include <cstdio>

#include "engine.h"
#include "kv_cache.cuh"
#include "kv_host.h"

namespace rtr {

constexpr int KV_THREADS = 256;

template <typename T> struct Dense;  // 16 bytes of a dense row
template <> struct Dense<float> {
  static constexpr int N = 4;
  static RTR_DEVICE void load(const float* p, float (&x)[4]) {
    const float4 u = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
  }
  static RTR_DEVICE void store(float* p, const float (&x)[4]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  }
};
template <> struct Dense<__nv_bfloat16> {
  static constexpr int N = 8;
  static RTR_DEVICE void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static RTR_DEVICE void store(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
};

// N codes of one thread (N = 4 or 8).
template <int N> struct Codes {
  uint32_t w[N / 4];
  RTR_DEVICE void load(const uint8_t* p) {
    if constexpr (N == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    }
  }
  RTR_DEVICE void store(uint8_t* p) const {
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
  RTR_DEVICE void get(float (&x)[N]) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t h = e4m3x2_to_f16x2((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
  RTR_DEVICE void set(const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      w[i] = (uint32_t)f32x2_to_e4m3x2(x[4 * i], x[4 * i + 1]) |
             ((uint32_t)f32x2_to_e4m3x2(x[4 * i + 2], x[4 * i + 3]) << 16);
  }
};

// The least power of two, from 2^-48 to 2^48, at which `amax` (at most 448 * 2^48)
// is at most 448 = 1.75 * 2^8: read off the float's exponent and mantissa.
RTR_DEVICE float least_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(127 + max(-KV_EXP, min(KV_EXP, e))) << 23);
}

// x / s, exactly rounded: by the reciprocal where s is a power of two (its
// reciprocal is one too), by a division for scales from elsewhere.
struct Divider {
  float s, r;
  bool pow2;
  explicit RTR_DEVICE Divider(float by) {
    s = by;
    r = 1.0f / by;
    pow2 = (__float_as_uint(by) & 0x7fffffu) == 0;
  }
  RTR_DEVICE float operator()(float x) const { return pow2 ? x * r : __fdiv_rn(x, s); }
};

// The part of a sequence's rows that falls into one of its pages.
struct PageRows {
  int page;       // page number
  int row0;       // the call's row of the page's token `lo`
  int lo, hi;     // tokens of the page that the call's rows fill
};

// Block `item` of a call: false where it has nothing to do.  Sequence b has the
// items from (starts[b] >> page_shift) + 2 b on: n rows from any token on touch at
// most floor(n / page) + 2 pages.
RTR_DEVICE bool kv_page_rows(const KvCache& c, const KvBatch& b, int64_t item, int per_seq, int* slot, PageRows& pr) {
  int seq;
  int64_t item0;
  if (b.starts) {
    seq = kv_find_seq(b, item, 1, c.page_shift, 2, slot, item0);
    if (seq < 0) return false;
  } else {
    seq = (int)(item / per_seq);
    item0 = (int64_t)seq * per_seq;
  }
  int first, count, len;
  if (!kv_rows(b, seq, 1, (int64_t)b.table_width << c.page_shift, c.status, first, count, len)) return false;
  const int begin = len - count;
  const int64_t nth = (begin >> c.page_shift) + (item - item0);
  const int64_t p0 = nth << c.page_shift;
  if (count == 0 || p0 >= len) return false;
  pr.lo = max(begin, (int)p0) - (int)p0;
  pr.hi = (int)(min((int64_t)len, p0 + (1 << c.page_shift)) - p0);
  pr.row0 = first + (int)p0 + pr.lo - begin;
  pr.page = kv_page(c, b, seq, (int)nth);
  return pr.page >= 0;
}

// CH 16-byte pieces of the page a thread: page * head_dim = CH * blockDim * N.
template <typename T, int CH>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const KvCache c, const KvBatch b, const T* __restrict__ k,
                                                              const T* __restrict__ v, const KvRows rs, int per_seq,
                                                              int units) {
  constexpr int N = Dense<T>::N;
  __shared__ int slot;
  __shared__ uint32_t red[2][KV_THREADS / 32];
  PageRows pr;
  if (!kv_page_rows(c, b, blockIdx.x, per_seq, &slot, pr)) return;
  const int tid = threadIdx.x, dpr = c.head_dim / N, warps = blockDim.x >> 5;
  const int u1 = min(2 * c.kv_heads, (int)(blockIdx.y + 1) * units);
  for (int u = blockIdx.y * units; u < u1; ++u) {
    const int head = u >> 1;
    const T* src = u & 1 ? v + head * rs.v_head : k + head * rs.k_head;
    const int64_t stride = u & 1 ? rs.v_token : rs.k_token;
    uint8_t* dst = (u & 1 ? c.v : c.k) + pr.page * c.page_stride + head * c.head_stride;
    float* scale = (u & 1 ? c.v_scale : c.k_scale) + pr.page * c.scale_stride + head;
    float x[CH][N];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / dpr;
      if (t >= pr.lo && t < pr.hi) {
        Dense<T>::load(src + (int64_t)(pr.row0 + t - pr.lo) * stride + (p % dpr) * N, x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[i][j] = 0.f;
      }
    }
    const float had = pr.lo > 0 ? *scale : 0.f;  // of the sequence's older tokens in this page
    // floats that are not negative order as their bits do
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float a = fabsf(x[i][j]);
        if (a <= 448.0f * 281474976710656.0f) top = max(top, __float_as_uint(a));
        else x[i][j] = __int_as_float(0x7fffffff);  // NaN, infinite or too large for the scales
      }
    top = __reduce_max_sync(0xffffffffu, top);
    uint32_t* r = red[u & 1];
    if ((tid & 31) == 0) r[tid >> 5] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = max(top, r[w]);
    float now = least_scale(__uint_as_float(top));
    if (pr.lo > 0) {
      if (!(had > 0.f && had < INFINITY)) {
        if (tid == 0) atomicOr(c.status, RTR_DEV_BAD_SCALE);
        continue;
      }
      now = fmaxf(now, had);
    }
    if (tid == 0 && now != had) *scale = now;
    const Divider over(now);
    const bool grown = pr.lo > 0 && now > had;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / dpr;
      Codes<N> q;
      if (t >= pr.lo && t < pr.hi) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[i][j] = over(x[i][j]);
        q.set(x[i]);
        q.store(dst + (int64_t)p * N);
      } else if (grown && t < pr.lo) {
        float y[N];
        q.load(dst + (int64_t)p * N);
        q.get(y);
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = over(y[j] * had);
        q.set(y);
        q.store(dst + (int64_t)p * N);
      }
    }
  }
}

template <typename T, int CH>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const KvCache c, const KvBatch b, T* __restrict__ k,
                                                             T* __restrict__ v, const KvRows rs, int per_seq,
                                                             int units) {
  constexpr int N = Dense<T>::N;
  __shared__ int slot;
  PageRows pr;
  if (!kv_page_rows(c, b, blockIdx.x, per_seq, &slot, pr)) return;
  const int tid = threadIdx.x, dpr = c.head_dim / N;
  const int u1 = min(2 * c.kv_heads, (int)(blockIdx.y + 1) * units);
  for (int u = blockIdx.y * units; u < u1; ++u) {
    const int head = u >> 1;
    T* dst = u & 1 ? v + head * rs.v_head : k + head * rs.k_head;
    const int64_t stride = u & 1 ? rs.v_token : rs.k_token;
    const uint8_t* src = (u & 1 ? c.v : c.k) + pr.page * c.page_stride + head * c.head_stride;
    const float scale = ((u & 1 ? c.v_scale : c.k_scale) + pr.page * c.scale_stride)[head];
    Codes<N> q[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / dpr;
      if (t >= pr.lo && t < pr.hi) q[i].load(src + (int64_t)p * N);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / dpr;
      if (t < pr.lo || t >= pr.hi) continue;
      float x[N];
      q[i].get(x);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= scale;
      Dense<T>::store(dst + (int64_t)(pr.row0 + t - pr.lo) * stride + (p % dpr) * N, x);
    }
  }
}

// ------------------------------------------------------------------- host
int kv_sms(int device, cudaError_t& e) {
  static std::atomic<int> known[64];
  if (device >= 0 && device < 64)
    if (const int n = known[device].load(std::memory_order_relaxed)) return n;
  int n = 0;
  e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess && device >= 0 && device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

const char* kv_check(const rtr_kv_cache* c, const rtr_kv_batch* b) {
  if (!c || !b) return "null cache or batch";
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->status) return "null cache buffer";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return "page must be 16, 32, 64 or 128 tokens";
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 16384) return "the cache needs pages and 1 to 16384 KV heads";
  if (c->head_stride < (int64_t)c->page * c->head_dim || c->page_stride < c->head_stride || c->scale_stride < 1)
    return "cache strides overlap";
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | (uintptr_t)c->page_stride |
       (uintptr_t)c->head_stride) & 15)
    return "codes and their strides must be multiples of 16 bytes";
  if (b->seqs < 0 || b->rows < 0) return "negative sequence or row count";
  if (b->seqs && (!b->lens || !b->table)) return "null table or lens";
  if (b->seqs && (b->table_width < 1 || b->table_stride < b->table_width)) return "table rows overlap or are empty";
  if ((int64_t)b->table_width * c->page > INT32_MAX - 4096) return "a table row holds at most 2^31 - 4096 tokens";
  if (!b->seqs && b->rows) return "rows without sequences";
  if (!b->starts && b->seqs && b->rows % b->seqs) return "rows must be a multiple of the sequences without starts";
  return nullptr;
}

KvCache kv_device_cache(const rtr_kv_cache* c) {
  int shift = 4;
  while ((1 << shift) < c->page) ++shift;
  return KvCache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, c->page_stride,
                 c->head_stride, c->scale_stride, c->pages, c->kv_heads, shift, c->head_dim, c->status};
}

KvBatch kv_device_batch(const rtr_kv_batch* b) {
  return KvBatch{b->table, b->lens, b->starts, b->table_stride, b->table_width, b->seqs, b->rows};
}

const char* kv_check_rows(const void* k, const void* v, int dtype, const KvRows& r, int head_dim) {
  const int size = dtype == RTR_DTYPE_F32 ? 4 : 2;
  if (dtype != RTR_DTYPE_F32 && dtype != RTR_DTYPE_BF16) return "dtype must be float32 or bfloat16";
  if (!k || !v) return "null rows";
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (uintptr_t)(r.k_token * size) |
       (uintptr_t)(r.k_head * size) | (uintptr_t)(r.v_token * size) | (uintptr_t)(r.v_head * size)) & 15)
    return "rows and their strides must be multiples of 16 bytes";
  return nullptr;
}

// Blocks of a write or read: page items, and how many units each block loops
// over.  Looping saves the walk to the page (starts, lens, table: ~2 us of latency)
// and costs parallelism: units are split while the grid is below eight blocks an SM.
KvGrid kv_page_grid(int rows, int seqs, bool starts, int page, int kv_heads, int sms) {
  KvGrid g;
  if (starts) {
    g.per_seq = 0;
    g.items = (int64_t)rows / page + 2 * (int64_t)seqs;
  } else {
    g.per_seq = (rows / seqs + page - 2) / page + 1;
    g.items = (int64_t)g.per_seq * seqs;
  }
  const int64_t all = 2 * (int64_t)kv_heads, want = 8 * (int64_t)sms;
  int64_t split = g.items >= want ? 1 : (want + g.items - 1) / g.items;
  if (split > all) split = all;
  g.units = (int)((all + split - 1) / split);
  g.splits = (int)((all + g.units - 1) / g.units);
  return g;
}

// Threads and 16-byte pieces a thread for a page of page * head_dim values.
template <typename T, typename F> static cudaError_t by_pieces(int values, F&& launch) {
  const int pieces = values / Dense<T>::N;
  if (pieces <= KV_THREADS) return launch(std::integral_constant<int, 1>{}, pieces);
  switch (pieces / KV_THREADS) {
    case 2: return launch(std::integral_constant<int, 2>{}, KV_THREADS);
    case 4: return launch(std::integral_constant<int, 4>{}, KV_THREADS);
    case 8: return launch(std::integral_constant<int, 8>{}, KV_THREADS);
    case 16: return launch(std::integral_constant<int, 16>{}, KV_THREADS);
  }
  return cudaErrorInvalidValue;
}

template <typename T, bool WRITE>
static cudaError_t launch_pages(const KvCache& c, const KvBatch& b, T* k, T* v, const KvRows& r, const KvGrid& g,
                                cudaStream_t stream) {
  return by_pieces<T>(c.head_dim << c.page_shift, [&](auto ch, int threads) {
    constexpr int CH = decltype(ch)::value;
    const dim3 grid((unsigned)g.items, (unsigned)g.splits);
    if constexpr (WRITE) kv_write_kernel<T, CH><<<grid, threads, 0, stream>>>(c, b, k, v, r, g.per_seq, g.units);
    else kv_read_kernel<T, CH><<<grid, threads, 0, stream>>>(c, b, k, v, r, g.per_seq, g.units);
    return cudaGetLastError();
  });
}

static int pages_call(bool write, const rtr_kv_cache* c, const rtr_kv_batch* b, void* k, void* v, int32_t dtype,
                      const KvRows& r, int32_t device, void* stream) {
  if (const char* e = kv_check(c, b)) return set_error(RTR_ERR_ARG, e);
  if (!b->rows) return RTR_OK;
  if (const char* e = kv_check_rows(k, v, dtype, r, c->head_dim)) return set_error(RTR_ERR_ARG, e);
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  const KvGrid g = kv_page_grid(b->rows, b->seqs, b->starts != nullptr, c->page, c->kv_heads, on.sms);
  if (g.items > INT32_MAX) return set_error(RTR_ERR_ARG, "too many rows and sequences for one call");
  const KvCache dc = kv_device_cache(c);
  const KvBatch db = kv_device_batch(b);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == RTR_DTYPE_F32) {
    float *kf = static_cast<float*>(k), *vf = static_cast<float*>(v);
    e = write ? launch_pages<float, true>(dc, db, kf, vf, r, g, st) : launch_pages<float, false>(dc, db, kf, vf, r, g, st);
  } else {
    auto *kh = static_cast<__nv_bfloat16*>(k), *vh = static_cast<__nv_bfloat16*>(v);
    e = write ? launch_pages<__nv_bfloat16, true>(dc, db, kh, vh, r, g, st)
              : launch_pages<__nv_bfloat16, false>(dc, db, kh, vh, r, g, st);
  }
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_kv_write(const rtr_kv_cache* cache, const rtr_kv_batch* batch, const void* k_dev, const void* v_dev,
                 int32_t dtype, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                 int64_t v_head_stride, int32_t device, void* stream) {
  return pages_call(true, cache, batch, const_cast<void*>(k_dev), const_cast<void*>(v_dev), dtype,
                    KvRows{k_token_stride, k_head_stride, v_token_stride, v_head_stride}, device, stream);
}

int rtr_kv_read(const rtr_kv_cache* cache, const rtr_kv_batch* batch, void* k_dev, void* v_dev, int32_t dtype,
                int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                int32_t device, void* stream) {
  return pages_call(false, cache, batch, k_dev, v_dev, dtype,
                    KvRows{k_token_stride, k_head_stride, v_token_stride, v_head_stride}, device, stream);
}

}  // extern "C"
