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
// thread.  Once a call has some thousand rows, reading is bound by HBM and writing by
// issue slots (77 % for 127,000 bf16 tokens of 4 heads, HBM 59 %): finding the maximum, scaling,
// rounding and packing are some 45 instructions for 8 values.  The write kernels hold a page's
// unit in registers and spill 16 - 52 bytes a thread at the limit that lets two or three blocks
// share an SM.
#include <cuda_runtime.h>

#include <cstdio>

#include "engine.h"
#include "kv_cache.cuh"
#include "kv_host.h"

namespace rtr {

constexpr int KV_THREADS = 512;
constexpr float KV_LARGEST = 448.0f * 281474976710656.0f;  // 448 * 2^48

// 16 bytes of a dense row, as they come and as values.
RTR_DEVICE uint4 load16(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }
RTR_DEVICE void values_of(const uint4& u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
RTR_DEVICE void values_of(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// The largest magnitude of 16 bytes of values, as a float's bits.
template <typename T> RTR_DEVICE uint32_t top_bits(const uint4& u);
template <> RTR_DEVICE uint32_t top_bits<float>(const uint4& u) {
  return max(max(u.x & 0x7fffffffu, u.y & 0x7fffffffu), max(u.z & 0x7fffffffu, u.w & 0x7fffffffu));
}
template <> RTR_DEVICE uint32_t top_bits<__nv_bfloat16>(const uint4& u) {
  const uint32_t m = 0x7fff7fffu, a = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  return max(a << 16, a & 0xffff0000u);
}
// The largest of all threads' values (one synchronisation; `red` is free again after the next).
RTR_DEVICE uint32_t block_max(uint32_t v, uint32_t* red, int warps) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0u);
}
RTR_DEVICE void store16(float* p, const float (&x)[4]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
}
RTR_DEVICE void store16(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}

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

// What the common path leaves: scales that are no power of two (from elsewhere; one float
// division, rounded, before the code is), values that become NaN; and older codes at a larger scale.
template <int N> __device__ __noinline__ Codes<N> encode_odd(uint4 raw, float s) {
  float x[N];
  values_of(raw, x);
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = fabsf(x[j]) <= KV_LARGEST ? __fdiv_rn(x[j], s) : __int_as_float(0x7fffffff);
  Codes<N> q;
  q.set(x);
  return q;
}
template <int N> __device__ __noinline__ Codes<N> encode_again(Codes<N> q, float had, float s) {
  float x[N];
  q.get(x);
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = __fdiv_rn(x[j] * had, s);
  q.set(x);
  return q;
}

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
    seq = kv_find_seq(b, item, 1, c.page_shift, 2, c.status, slot, item0);
    if (seq < 0) return false;
  } else {
    seq = (int)(item / per_seq);
    item0 = (int64_t)seq * per_seq;
  }
  int first, count;
  const int len = b.lens[seq];
  if (!kv_rows(b, seq, c.status, first, count) || !kv_len_fits(c, b, len, count)) return false;
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

// A block's threads take CH 16-byte pieces of the page each: page * D = CH * blockDim * N.
// AHEAD: the next unit's rows are on their way while a unit's maximum is found and its
// codes are written.  Blocks of one unit are without, in registers that let three of 512
// threads share an SM (two with eight pieces): 350 fp32 tokens of 56 heads, 13.0 us with
// the registers of AHEAD, 9.4 us without.
template <typename T, int D, int CH, bool AHEAD>
__global__ void __launch_bounds__(KV_THREADS, CH == 4 && !AHEAD ? 3 : 2) kv_write_kernel(const KvCache c, const KvBatch b, const T* k,
                                                              const T* v, const KvRows rs, int per_seq,
                                                              int units) {
  constexpr int N = 16 / sizeof(T), DPR = D / N;  // values of a piece, pieces of a row
  __shared__ int slot[2];
  __shared__ uint32_t red[2][KV_THREADS / 32];
  PageRows pr;
  pdl_launch_dependents();
  pdl_wait();
  if (!kv_page_rows(c, b, blockIdx.x, per_seq, slot, pr)) return;
  const int tid = threadIdx.x, warps = blockDim.x >> 5;
  const int u0 = blockIdx.y * units, u1 = min(2 * c.kv_heads, u0 + units);
  const bool kept = pr.lo > 0;  // the page holds older tokens of the sequence
  const auto scale_of = [&](int u) { return (u & 1 ? c.v_scale : c.k_scale) + pr.page * c.scale_stride + (u >> 1); };
  const auto load = [&](int u, uint4 (&raw)[CH], float& had) {
    const T* src = u & 1 ? v + (u >> 1) * rs.v_head : k + (u >> 1) * rs.k_head;
    const int64_t stride = u & 1 ? rs.v_token : rs.k_token;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / DPR;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (t >= pr.lo && t < pr.hi) raw[i] = load16(src + (int64_t)(pr.row0 + t - pr.lo) * stride + (p % DPR) * N);
    }
    had = kept ? *scale_of(u) : 0.f;
  };
  uint4 raw[CH], next[AHEAD ? CH : 1];
  float had, next_had = 0.f;
  load(u0, raw, had);
  for (int u = u0; u < u1; ++u) {
    if constexpr (AHEAD)
      if (u + 1 < u1) load(u + 1, next, next_had);
    uint8_t* dst = (u & 1 ? c.v : c.k) + pr.page * c.page_stride + (u >> 1) * c.head_stride;
    // Magnitudes order as their bits do.  A unit whose largest bits are those of a NaN, an
    // infinite or a too large value is looked through again without them.
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) top = max(top, top_bits<T>(raw[i]));
    top = block_max(top, red[u & 1], warps);
    const bool odd = top > __float_as_uint(KV_LARGEST);
    if (odd) {
      top = 0;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float x[N];
        values_of(raw[i], x);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (fabsf(x[j]) <= KV_LARGEST) top = max(top, __float_as_uint(fabsf(x[j])));
      }
      __syncthreads();  // every warp has read the first maximum
      top = block_max(top, red[u & 1], warps);
    }
    float now = least_scale(__uint_as_float(top));
    const bool fits = !kept || (had > 0.f && had < INFINITY);
    if (!fits) {
      if (tid == 0) atomicOr(c.status, RTR_DEV_BAD_SCALE);
    } else {
      if (kept) now = fmaxf(now, had);
      if (tid == 0 && now != had) *scale_of(u) = now;
      // a power of two has an exact reciprocal
      const float inverse = 1.0f / now;
      const bool plain = !odd && (__float_as_uint(now) & 0x7fffffu) == 0;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int p = tid + i * blockDim.x, t = p / DPR;
        if (t < pr.lo || t >= pr.hi) continue;
        Codes<N> q;
        if (plain) {
          float x[N];
          values_of(raw[i], x);
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] *= inverse;
          q.set(x);
        } else {
          q = encode_odd<N>(raw[i], now);
        }
        q.store(dst + (int64_t)p * N);
      }
      if (kept && now > had) {
        for (int p = tid; p < pr.lo * DPR; p += blockDim.x) {
          Codes<N> q;
          q.load(dst + (int64_t)p * N);
          encode_again<N>(q, had, now).store(dst + (int64_t)p * N);
        }
      }
    }
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < CH; ++i) raw[i] = next[i];
      had = next_had;
    } else if (u + 1 < u1) {
      load(u + 1, raw, had);
    }
  }
}

template <typename T, int D, int CH>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const KvCache c, const KvBatch b, T* k,
                                                             T* v, const KvRows rs, int per_seq,
                                                             int units) {
  constexpr int N = 16 / sizeof(T), DPR = D / N;
  __shared__ int slot[2];
  PageRows pr;
  pdl_launch_dependents();
  pdl_wait();
  if (!kv_page_rows(c, b, blockIdx.x, per_seq, slot, pr)) return;
  const int tid = threadIdx.x;
  const int u0 = blockIdx.y * units, u1 = min(2 * c.kv_heads, u0 + units);
  const auto load = [&](int u, Codes<N> (&q)[CH], float& scale) {
    const uint8_t* src = (u & 1 ? c.v : c.k) + pr.page * c.page_stride + (u >> 1) * c.head_stride;
    scale = ((u & 1 ? c.v_scale : c.k_scale) + pr.page * c.scale_stride)[u >> 1];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / DPR;
      if (t >= pr.lo && t < pr.hi) q[i].load(src + (int64_t)p * N);
    }
  };
  Codes<N> q[CH], next[CH];
  float scale, next_scale = 0.f;
  load(u0, q, scale);
  for (int u = u0; u < u1; ++u) {
    if (u + 1 < u1) load(u + 1, next, next_scale);
    T* dst = u & 1 ? v + (u >> 1) * rs.v_head : k + (u >> 1) * rs.k_head;
    const int64_t stride = u & 1 ? rs.v_token : rs.k_token;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = tid + i * blockDim.x, t = p / DPR;
      if (t < pr.lo || t >= pr.hi) continue;
      float x[N];
      q[i].get(x);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= scale;
      store16(dst + (int64_t)(pr.row0 + t - pr.lo) * stride + (p % DPR) * N, x);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) q[i] = next[i];
    scale = next_scale;
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
  const int64_t one = (int64_t)c->page * c->head_dim;  // codes of a page's head
  if (c->head_stride < one || c->page_stride < one || c->scale_stride < c->kv_heads) return "cache strides overlap";
  // the heads of a page before the next page, or the pages of a head before the next head
  if (c->kv_heads > 1 && (c->page_stride - one) / (c->kv_heads - 1) < c->head_stride &&
      c->pages > 1 && (c->head_stride - one) / (c->pages - 1) < c->page_stride)
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

// Threads and 16-byte pieces a thread for a page of `pieces` (a power of two from 128 to
// 4096): four pieces a thread spread a unit's fixed work (maximum, scale, addresses)
// and leave registers for the next unit's.
template <typename F> static cudaError_t by_pieces(int pieces, F&& launch) {
  if (pieces <= 4 * KV_THREADS) return launch(std::integral_constant<int, 4>{}, pieces / 4);
  return launch(std::integral_constant<int, 8>{}, pieces / 8);
}

template <typename T, int D, bool WRITE>
static cudaError_t launch_pages(const KvCache& c, const KvBatch& b, T* k, T* v, const KvRows& r, const KvGrid& g,
                                cudaStream_t stream) {
  return by_pieces((D << c.page_shift) * (int)sizeof(T) / 16, [&](auto ch, int threads) {
    constexpr int CH = decltype(ch)::value;
    const dim3 grid((unsigned)g.items, (unsigned)g.splits);
    const auto run = [&](auto kernel) { return kv_launch(kernel, grid, threads, 0, 1, stream, c, b, k, v, r, g.per_seq, g.units); };
    if constexpr (!WRITE) return run(kv_read_kernel<T, D, CH>);
    else if (CH == 4 && g.units > 1) return run(kv_write_kernel<T, D, CH, CH == 4>);
    else return run(kv_write_kernel<T, D, CH, false>);
  });
}

template <typename T>
static cudaError_t launch_pages(bool write, const KvCache& c, const KvBatch& b, void* k, void* v, const KvRows& r,
                                const KvGrid& g, cudaStream_t st) {
  T *kt = static_cast<T*>(k), *vt = static_cast<T*>(v);
  if (c.head_dim == 128)
    return write ? launch_pages<T, 128, true>(c, b, kt, vt, r, g, st) : launch_pages<T, 128, false>(c, b, kt, vt, r, g, st);
  return write ? launch_pages<T, 64, true>(c, b, kt, vt, r, g, st) : launch_pages<T, 64, false>(c, b, kt, vt, r, g, st);
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
  const cudaError_t e = dtype == RTR_DTYPE_F32 ? launch_pages<float>(write, dc, db, k, v, r, g, st)
                                               : launch_pages<__nv_bfloat16>(write, dc, db, k, v, r, g, st);
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
