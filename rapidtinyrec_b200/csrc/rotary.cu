// Rotary positions: pairs of dimensions of q and k turned by angles that grow with the position.
//
// Mathematics.  A frequency is kept as 64 bits of turns a position, so the angle of position p is
// the product p * turns modulo 2^64: integer arithmetic drops the whole turns and keeps the rest
// exactly, at position 2^31 as at 1, where an fp32 angle of position 130,000 is off by
// 0.004 radians.  Its upper 32 bits, taken as a signed fraction of a turn, go to sincospif.
//
// What bounds it: q and k are read and written once, so HBM for many rows (and for few the launch and
// two dependent loads, the position and the angles' end of the chain).  A row's angles are
// the same for every head: a thread keeps the sines and cosines of its pairs in registers (8 pairs in bf16, 4 in
// fp32: two 16-byte pieces) and goes over several heads with them.  One sincospif costs some 30 instructions;
// over four heads that is 1.9 of the 5.5 instructions a byte that the SMs issue while HBM delivers it.  27,009 rows of 28/4 heads of 128,
// bf16: 70.4 us, 6.3 TB/s, 97 % of the copy rate (with the values unpacked as they were loaded, 114 registers
// instead of 80, 121 us); one row of 12/2 heads, fp32, 1.9 us on the device.
#include <cuda_runtime.h>

#include <type_traits>

#include "engine.h"
#include "kv_host.h"

namespace rtr {

constexpr int RO_THREADS = 256, RO_HEADS = 4;  // heads a thread has in flight

struct RotaryRows {
  const void* in;
  void* out;
  int64_t in_row, in_head, out_row, out_head;
};

struct Rotary {
  RotaryRows q, k;
  int64_t rows;
  const void* positions;
  const uint64_t* turns;
  float factor, sign;
  int q_heads, heads;       // of q, of both
  int half, units, turned;  // pairs of a head; pieces of a head, and those of them that turn
  int rest, dim;            // first dimension of the pieces that are only copied; dimensions of a head
  int split, per_block;     // threads that share a row's heads, rows of a block
  bool wide;
};

// N values of a thread's piece, as they lie in memory: 16 bytes, or one value where rows do not lie at multiples of 16.
template <typename T, int N> struct Piece {
  using Raw = typename std::conditional<N == 1, T, uint4>::type;
  Raw u;
  RTR_DEVICE void load(const T* p) { u = *reinterpret_cast<const Raw*>(p); }
  RTR_DEVICE void get(float (&x)[N]) const {
    if constexpr (N == 1) {
      x[0] = to_f32(u);
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (N == 4) {
          x[i] = __uint_as_float(w[i]);
        } else {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
  RTR_DEVICE void set(const float (&x)[N]) {
    if constexpr (N == 1) {
      u = from_f32<T>(x[0]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (N == 4) {
          w[i] = __float_as_uint(x[i]);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      u = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  RTR_DEVICE void store(T* p) const { *reinterpret_cast<Raw*>(p) = u; }
};

RTR_DEVICE void turn(float& a, float& b, float cosine, float sine) {
  const float u = a;
  a = fmaf(u, cosine, -b * sine);
  b = fmaf(b, cosine, u * sine);
}

template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(const Rotary a) {
  const int tid = threadIdx.x, span = a.units * a.split, in_block = tid / span;
  const int64_t row = (int64_t)blockIdx.x * a.per_block + in_block;
  pdl_launch_dependents();
  pdl_wait();
  if (in_block >= a.per_block || row >= a.rows) return;
  const int left = tid - in_block * span, first = left / a.units, unit = left - first * a.units;
  const bool turns = unit < a.turned;
  // the thread's two pieces: the two sides of N pairs, or 2 N neighbouring dimensions
  int d0, d1;
  if (!turns) {
    d0 = a.rest + 2 * N * (unit - a.turned);
    d1 = d0 + N;
  } else if constexpr (INTERLEAVED) {
    d0 = 2 * N * unit;
    d1 = d0 + N;
  } else {
    d0 = N * unit;
    d1 = d0 + a.half;
  }
  const bool second = N > 1 || turns || d1 < a.dim;  // an odd last dimension has no neighbour
  float cosine[N], sine[N];
  bool known = false;
  for (int h0 = first; h0 < a.heads; h0 += RO_HEADS * a.split) {
    Piece<T, N> x[RO_HEADS], y[RO_HEADS];
#pragma unroll
    for (int j = 0; j < RO_HEADS; ++j) {
      const int h = h0 + j * a.split;
      if (h >= a.heads) continue;
      const RotaryRows& r = h < a.q_heads ? a.q : a.k;
      const T* p = static_cast<const T*>(r.in) + row * r.in_row + (int64_t)(h < a.q_heads ? h : h - a.q_heads) * r.in_head;
      x[j].load(p + d0);
      if (second) y[j].load(p + d1);
    }
    if (!known && turns) {
      const int64_t position = a.wide ? static_cast<const int64_t*>(a.positions)[row] : static_cast<const int32_t*>(a.positions)[row];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint64_t t = (uint64_t)position * a.turns[N * unit + i];
        sincospif((float)(int32_t)(t >> 32) * 4.656612873077393e-10f, &sine[i], &cosine[i]);  // 2^-31: half turns
        sine[i] *= a.factor * a.sign;
        cosine[i] *= a.factor;
      }
      known = true;
    }
#pragma unroll
    for (int j = 0; j < RO_HEADS; ++j) {
      const int h = h0 + j * a.split;
      if (h >= a.heads) continue;
      if (turns) {
        float u[N], v[N];
        x[j].get(u);
        y[j].get(v);
        if constexpr (INTERLEAVED && N > 1) {
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            turn(u[2 * i], u[2 * i + 1], cosine[i], sine[i]);
            turn(v[2 * i], v[2 * i + 1], cosine[N / 2 + i], sine[N / 2 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) turn(u[i], v[i], cosine[i], sine[i]);
        }
        x[j].set(u);
        y[j].set(v);
      }
      const RotaryRows& r = h < a.q_heads ? a.q : a.k;
      T* p = static_cast<T*>(r.out) + row * r.out_row + (int64_t)(h < a.q_heads ? h : h - a.q_heads) * r.out_head;
      x[j].store(p + d0);
      if (second) y[j].store(p + d1);
    }
  }
}

static const char* rotary_check(const rtr_rotary_rows* r, int64_t rows, int head_dim) {
  if (r->heads < 1) return "rows need heads";
  if (rows && (!r->in || !r->out)) return "null rows";
  if (r->out_head < head_dim && r->heads > 1) return "heads of the output overlap";
  if (rows > 1 && r->out_row < head_dim) return "rows of the output overlap";
  if (r->in == r->out && ((rows > 1 && r->in_row != r->out_row) || (r->heads > 1 && r->in_head != r->out_head)))
    return "rows turned in place need one set of strides";
  return nullptr;
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_rotary(const rtr_rotary_rows* q, const rtr_rotary_rows* k, int64_t rows, int32_t head_dim, int32_t rotary_dim,
               int32_t interleaved, int32_t dtype, const void* positions, int32_t wide, const uint64_t* turns, float factor,
               int32_t back, int32_t device, void* stream) {
  if (!q) return set_error(RTR_ERR_ARG, "null rows");
  if (dtype != RTR_DTYPE_F32 && dtype != RTR_DTYPE_BF16) return set_error(RTR_ERR_ARG, "dtype must be float32 or bfloat16");
  if (head_dim < 2 || head_dim > 512 || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return set_error(RTR_ERR_ARG, "head_dim must be 2 to 512 and rotary_dim even and at most head_dim");
  if (rows < 0) return set_error(RTR_ERR_ARG, "negative row count");
  if (const char* e = rotary_check(q, rows, head_dim)) return set_error(RTR_ERR_ARG, e);
  if (k)
    if (const char* e = rotary_check(k, rows, head_dim)) return set_error(RTR_ERR_ARG, e);
  if (!rows) return RTR_OK;
  if (!positions || !turns) return set_error(RTR_ERR_ARG, "null positions or turns");
  const int size = dtype == RTR_DTYPE_F32 ? 4 : 2, wide_n = 16 / size;
  uintptr_t bits = 0;
  bool in_place = true;
  for (const rtr_rotary_rows* r : {q, k}) {
    if (!r) continue;
    bits |= reinterpret_cast<uintptr_t>(r->in) | reinterpret_cast<uintptr_t>(r->out);
    if (rows > 1) bits |= (uintptr_t)((r->in_row | r->out_row) * size);
    if (r->heads > 1) bits |= (uintptr_t)((r->in_head | r->out_head) * size);
    in_place = in_place && r->in == r->out;
  }
  const int rest = in_place ? 0 : head_dim - rotary_dim;
  const bool pieces = bits % 16 == 0 && rotary_dim % (2 * wide_n) == 0 && rest % (2 * wide_n) == 0;
  const int n = pieces ? wide_n : 1;
  Rotary a = {};
  const auto put = [](RotaryRows& to, const rtr_rotary_rows* r) {
    to = RotaryRows{r->in, r->out, r->in_row, r->in_head, r->out_row, r->out_head};
  };
  put(a.q, q);
  if (k) put(a.k, k);
  a.rows = rows;
  a.positions = positions;
  a.turns = turns;
  a.factor = factor;
  a.sign = back ? -1.f : 1.f;
  a.q_heads = q->heads;
  a.heads = q->heads + (k ? k->heads : 0);
  a.half = rotary_dim / 2;
  a.turned = rotary_dim / (2 * n);
  a.units = a.turned + (rest + 2 * n - 1) / (2 * n);
  a.rest = rotary_dim;
  a.dim = head_dim;
  a.wide = wide != 0;
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  // Threads that share a row's heads: all that fit a block while there are few rows, and four heads a thread
  // where the rows alone fill the GPU's threads twice.
  const int64_t full = 2 * 2048 * (int64_t)on.sms;
  int split = RO_THREADS / a.units;
  if (split > a.heads) split = a.heads;
  const int few = (a.heads + RO_HEADS - 1) / RO_HEADS;
  if (split > few && rows * a.units * few >= full) split = few;
  a.split = split < 1 ? 1 : split;
  a.per_block = RO_THREADS / (a.units * a.split);
  const int64_t blocks = (rows + a.per_block - 1) / a.per_block;
  if (blocks > INT32_MAX) return set_error(RTR_ERR_ARG, "too many rows for one call");
  const auto launch = [&](auto kernel) {
    return kv_launch(kernel, dim3((unsigned)blocks), RO_THREADS, 0, 1, static_cast<cudaStream_t>(stream), a);
  };
  cudaError_t e;
  if (dtype == RTR_DTYPE_F32) {
    if (pieces) e = interleaved ? launch(rotary_kernel<float, 4, true>) : launch(rotary_kernel<float, 4, false>);
    else e = interleaved ? launch(rotary_kernel<float, 1, true>) : launch(rotary_kernel<float, 1, false>);
  } else {
    if (pieces) e = interleaved ? launch(rotary_kernel<__nv_bfloat16, 8, true>) : launch(rotary_kernel<__nv_bfloat16, 8, false>);
    else e = interleaved ? launch(rotary_kernel<__nv_bfloat16, 1, true>) : launch(rotary_kernel<__nv_bfloat16, 1, false>);
  }
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
