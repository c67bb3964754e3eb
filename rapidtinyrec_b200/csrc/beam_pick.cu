// The best continuations of beams over the whole vocabulary, from one pass over the logits.
//
// Mathematics.  Candidate (i, v) is worth x[i][v] - lse[i] + score[i] with lse the log of the sum
// of exponentials of row i.  Within a row the order is that of the logits; across rows it
// needs lse, which is known only when a row has been read.  So the first kernel
// reads each logit once and leaves, beside the row's running maximum and sum, the largest logit of every
// group of 256.  The k-th largest of the groups' best is a lower bound T of the k-th largest candidate, and only
// groups whose best reaches T can hold one of the k: k of them but for ties.  The second kernel
// (a block an item) finds T, reads those groups again (25,600 of 7.6 million logits for 100 candidates of 50 beams), takes what
// reaches T and puts it in order.
//
// Order.  The sums are fp32 (an error of some 2e-7 in lse), the 100 best of 7.6 million candidates lie 1e-3 apart, and a batch
// has thousands of neighbours, so now and then two are too close to tell.  Differences of logits and scores are exact
// enough in fp64; what is not known well is lse.  Where two neighbours of different rows are closer than
// BP_DOUBT, both rows' sums are taken again in fp64 and the list is put in order again: the result
// is what 64-bit arithmetic gives, whatever the split of the rows.
//
// What bounds it: the first kernel HBM (4.5 instructions and one exponential a logit, of 11 and 1.4 that the SMs issue while bf16
// logits arrive), the second latency: three dependent rounds of loads and the searches between them.
#include <cuda_runtime.h>

#include <type_traits>

#include "engine.h"
#include "kv_attention.cuh"
#include "kv_host.h"

namespace rtr {

constexpr int BP_GROUP = 256;                   // logits of a group: eight of each lane of a warp
constexpr int BP_WARPS = 8, BP_AHEAD = 4;       // first kernel: warps of a block, groups a warp has in flight
constexpr int BP_THREADS = 1024;                // second kernel
constexpr int BP_MAX_N = 128, BP_MAX_K = 256;
constexpr int BP_GROUPS = 512, BP_LIST = 1024;  // groups and candidates that the second kernel takes up at once
constexpr double BP_DOUBT = 1e-6;               // candidates of different rows that are closer are looked at again
constexpr float BP_LOG2E = 1.4426950408889634f;

struct BeamPick {
  const void* logits;
  const float* scores;
  const uint8_t* allowed;
  int64_t stride, allowed_stride;
  int items, n, vocab, k, beams, eos;
  int groups, padded;      // groups of a row, and their number rounded up to 4
  uint32_t quarter_inv;    // ceil(2^32 / (padded / 4)): a group quartet's row by one multiplication (0: 2^32, the quartet itself)
  int slices;              // blocks of a row
  float* best;             // [items * n][padded]: a group's largest allowed logit
  float2* part;            // [items * n][slices]: maximum, sum of exponentials relative to it
  int32_t *all_tokens, *all_parents, *next_tokens, *next_parents;
  float *all_scores, *next_scores;
  uint32_t* status;
};

RTR_DEVICE float redux_max(float v) {  // NaN counts as nothing
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// A warp's part of a group: each lane has eight logits, in pieces of 16 bytes.  Groups start at multiples
// of 16 bytes: the first of a row that does not holds fewer.
template <typename T> struct Logits {
  static constexpr int PER = 16 / sizeof(T), PIECES = 8 / PER;
  uint4 u[PIECES];
  RTR_DEVICE static int shift(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
  RTR_DEVICE static int at(int first, int i, int lane) { return first + (i / PER) * 32 * PER + lane * PER + i % PER; }
  RTR_DEVICE void none() {
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) u[j] = make_uint4(w, w, w, w);
  }
  RTR_DEVICE void load(const T* row, int first, int lane, int vocab) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int e = at(first, j * PER, lane);
      if (e >= 0 && e + PER <= vocab) {
        u[j] = __ldg(reinterpret_cast<const uint4*>(row + e));
      } else {  // a row's ragged ends
        const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xff80u;
        uint32_t v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          v[i] = w;
          if (e + i >= 0 && e + i < vocab) {
            if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(row[e + i]);
            else v[i] = __bfloat16_as_ushort(row[e + i]);
          }
        }
        if constexpr (sizeof(T) == 4) u[j] = make_uint4(v[0], v[1], v[2], v[3]);
        else u[j] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
      }
    }
  }
  RTR_DEVICE void get(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          x[4 * j + i] = __uint_as_float(w[i]);
        } else {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
};

// Which of a lane's eight logits are allowed, as bits.  Four bytes at a time, by aligned words that hold
// at least one of them, since a row of bytes may start anywhere.
template <typename T> RTR_DEVICE uint32_t allowed_bits(const uint8_t* row, int first, int lane, int vocab) {
  using L = Logits<T>;
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = L::at(first, 4 * j, lane);
    uint32_t four = 0;
    if (e >= 0 && e + 4 <= vocab) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(row + e);
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p & ~(uintptr_t)3);
      const int by = (int)(p & 3);
      four = __ldg(w);
      if (by) four = __funnelshift_r(four, __ldg(w + 1), 8 * by);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i >= 0 && e + i < vocab) four |= (uint32_t)row[e + i] << (8 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= (four >> (8 * i) & 0xffu ? 1u : 0u) << (4 * j + i);
  }
  return bits;
}

// One block: a slice of a row's groups.
template <typename T, bool MASK>
__global__ void __launch_bounds__(BP_WARPS * 32, 4) beam_scan_kernel(const BeamPick a) {
  __shared__ float2 sums[BP_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const float score = a.scores[row];
  if (!(score > -INFINITY)) {  // minus infinity: nothing to offer; NaN: the second kernel reports it
    if (tid == 0) a.part[blockIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const uint8_t* allowed = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  const int shift = Logits<T>::shift(x);
  const int lo = (int)((int64_t)a.groups * slice / a.slices), hi = (int)((int64_t)a.groups * (slice + 1) / a.slices);
  if (slice == a.slices - 1 && tid < a.padded - a.groups) a.best[(int64_t)row * a.padded + a.groups + tid] = -INFINITY;
  float base = -INFINITY;
  uint64_t sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
  const uint64_t log2e = f2(BP_LOG2E, BP_LOG2E);
  for (int g = lo + warp * BP_AHEAD; g < hi; g += BP_WARPS * BP_AHEAD) {
    Logits<T> raw[BP_AHEAD];
    uint32_t bits[BP_AHEAD];
#pragma unroll
    for (int j = 0; j < BP_AHEAD; ++j) {
      const int first = (g + j) * BP_GROUP - shift;
      if (g + j < hi) raw[j].load(x, first, lane, a.vocab);
      else raw[j].none();
      if constexpr (MASK) bits[j] = g + j < hi ? allowed_bits<T>(allowed, first, lane, a.vocab) : 0u;
    }
    float top = -INFINITY, mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < BP_AHEAD; ++j) {
      float v[8], m = -INFINITY;
      raw[j].get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, v[i]);
      m = redux_max(m);
      top = fmaxf(top, m);
      if constexpr (MASK) {
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, bits[j] >> i & 1 ? v[i] : -INFINITY);
        m = redux_max(m);
      }
      if (lane == j) mine = m;
    }
    if (lane < BP_AHEAD && g + lane < hi) a.best[(int64_t)row * a.padded + g + lane] = mine;
    if (top > base) {  // the same in all lanes
      const float f = ex2((base - top) * BP_LOG2E);
#pragma unroll
      for (int i = 0; i < 2; ++i) sum[i] = f2_mul(sum[i], f2(f, f));
      base = top;
    }
    const float zero = base == -INFINITY ? 0.f : -base;
    const uint64_t minus = f2(zero, zero);
#pragma unroll
    for (int j = 0; j < BP_AHEAD; ++j) {
      float v[8];
      raw[j].get(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = f2_parts(f2_mul(f2_add(f2(v[2 * i], v[2 * i + 1]), minus), log2e));
        sum[i & 1] = f2_add(sum[i & 1], f2(ex2(y.x), ex2(y.y)));
      }
    }
  }
  const float2 s = f2_parts(f2_add(sum[0], sum[1]));
  const float total = warp_sum(s.x + s.y);
  if (lane == 0) sums[warp] = make_float2(base, total);
  __syncthreads();
  if (tid == 0) {
    float m = -INFINITY, t = 0.f;
#pragma unroll
    for (int w = 0; w < BP_WARPS; ++w) m = fmaxf(m, sums[w].x);
#pragma unroll
    for (int w = 0; w < BP_WARPS; ++w) t += sums[w].x == m ? sums[w].y : sums[w].y * ex2((sums[w].x - m) * BP_LOG2E);
    a.part[blockIdx.x] = make_float2(m, t);
  }
}

// ------------------------------------------------------------ second kernel
// Order-preserving map double -> uint64.
RTR_DEVICE uint64_t double_key(double d) {
  const uint64_t u = (uint64_t)__double_as_longlong(d);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
RTR_DEVICE double key_double(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

struct PickShared {
  double sum[BP_MAX_N], off[BP_MAX_N];  // log of the sum of exponentials relative to the maximum, score - that
  float off32[BP_MAX_N], top[BP_MAX_N];  // off rounded (minus infinity: nothing to offer), the row's maximum
  uint8_t again[BP_MAX_N], done[BP_MAX_N];  // rows to sum in 64 bits, and those that are
  int32_t groups[BP_GROUPS];
  uint64_t key[BP_LIST];
  float x[BP_LIST];
  uint32_t at[BP_LIST];
  uint16_t order[BP_LIST];
  double red[BP_THREADS / 32];
  int n_groups, n_list, doubts;
  float most;
};

// A value that at least k threads reach with what they have, or minus infinity where fewer have a finite one:
// bit by bit from the top of the keys, until the count is near k.
RTR_DEVICE float reached_by(float mine, int k) {
  const uint32_t key = mine > -INFINITY ? float_key(mine) : 0u;
  uint32_t low = 0;
  const int near = k + (k >> 3) + 4;
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = low | 1u << b;
    const int c = __syncthreads_count(key >= t);
    if (c < k) continue;
    low = t;
    if (c <= near) break;
  }
  return low ? key_float(low) : -INFINITY;
}

template <typename T, bool MASK> struct Picker {
  const BeamPick& a;
  PickShared& s;
  const int item, tid, warp, lane;
  const T* x0;               // the item's first row
  const uint8_t* allowed0;
  const float* best;         // [n][padded]

  RTR_DEVICE int row_of(uint32_t quartet) const { return (int)(a.quarter_inv ? __umulhi(quartet, a.quarter_inv) : quartet); }
  RTR_DEVICE const T* row(int r) const { return x0 + r * a.stride; }
  // what a candidate is worth, and nearly so
  RTR_DEVICE double worth(int r, float x) const { return ((double)x - (double)s.top[r]) + s.off[r]; }
  RTR_DEVICE float near(int r, float x) const { return (x - s.top[r]) + s.off32[r]; }

  // f(group index row * padded + g, best logit) for the thread's groups, of rows that are alive
  template <typename F> RTR_DEVICE void each_group(F&& f) const {
    const int quartets = a.padded >> 2, all = a.n * quartets;
    for (int q = tid; q < all; q += BP_THREADS) {
      const int r = a.n == 1 ? 0 : row_of((uint32_t)q);
      if (!(s.off32[r] > -INFINITY)) continue;
      const float4 v = __ldcg(reinterpret_cast<const float4*>(best) + q);
      const int g0 = 4 * (q - r * quartets);
      f(r, g0, v);
    }
  }

  // f(row, place in the vocabulary, logit) for a lane's allowed logits of group r, g
  template <typename F> RTR_DEVICE void each_logit(int r, int g, const Logits<T>& raw, uint32_t bits, F&& f) const {
    float v[8];
    raw.get(v);
    const int first = g * BP_GROUP - Logits<T>::shift(row(r));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i] > -INFINITY && (!MASK || (bits >> i & 1))) f(r, Logits<T>::at(first, i, lane), v[i]);
  }

  // Each row's sum from its slices, and what its candidates are offset by
  RTR_DEVICE void offsets() {
    for (int r = warp; r < a.n; r += BP_THREADS / 32) {
      const float2* p = a.part + ((int64_t)item * a.n + r) * a.slices;
      float m = -INFINITY;
      for (int i = lane; i < a.slices; i += 32) m = fmaxf(m, __ldcg(&p[i].x));
      m = redux_max(m);
      double t = 0.0;
      for (int i = lane; i < a.slices; i += 32) {
        const float2 v = __ldcg(p + i);
        t += v.x == m ? (double)v.y : (double)v.y * exp((double)v.x - (double)m);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      if (lane == 0) {
        const float score = a.scores[item * a.n + r];
        const bool wrong = !(score < INFINITY) || (score > -INFINITY && !(t >= 0.0 && m < INFINITY));
        if (wrong) atomicOr(a.status, RTR_DEV_NAN_SCORE);
        const bool alive = !wrong && score > -INFINITY && m > -INFINITY;
        s.sum[r] = alive ? log(t) : 0.0;
        s.top[r] = m;
        s.off[r] = alive ? (double)score - s.sum[r] : -INFINITY;
        s.off32[r] = (float)s.off[r];
        s.again[r] = s.done[r] = 0;
      }
    }
    __syncthreads();
    if (warp == 0) {
      float most = 0.f;
      for (int r = lane; r < a.n; r += 32)
        if (s.off32[r] > -INFINITY) most = fmaxf(most, fabsf(s.off32[r]));
      most = redux_max(most);
      if (lane == 0) s.most = most;
    }
    __syncthreads();
  }

  // The sums of the rows marked `again`, in 64 bits: one row after the other, all threads.  The order of
  // a sum goes by places in the vocabulary, not by the row's place in memory, so that equal rows have equal sums.
  RTR_DEVICE void sum_again() {
    for (int r = 0; r < a.n; ++r) {
      if (!s.again[r] || s.done[r]) continue;  // the same for all threads
      const T* p = row(r);
      const double m = s.top[r];
      double t = 0.0;
      for (int i0 = tid; i0 < a.vocab; i0 += 8 * BP_THREADS) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i0 + i * BP_THREADS < a.vocab ? to_f32(p[i0 + i * BP_THREADS]) : -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double d = (double)v[i] - m;
          if (d > -100.0) t += exp(d);  // a vocabulary of what is left out is below 2^-124 of the sum
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      if (lane == 0) s.red[warp] = t;
      __syncthreads();
      if (tid == 0) {
        t = 0.0;
        for (int w = 0; w < BP_THREADS / 32; ++w) t += s.red[w];
        s.sum[r] = log(t);
        s.off[r] = (double)a.scores[item * a.n + r] - s.sum[r];
        s.off32[r] = (float)s.off[r];
        s.done[r] = 1;
      }
      __syncthreads();
    }
  }

  // What `near` may be off by (three roundings of 2^-24), with room, and what two sums may be.
  RTR_DEVICE float slack(float t) const { return (float)BP_DOUBT + 4.77e-7f * (s.most + fabsf(t)); }

  // The groups and then the candidates that reach the k-th best of what stands for them: false where there are too
  // many (ties).
  RTR_DEVICE bool gather() {
    if (tid == 0) s.n_groups = s.n_list = 0;
    float mine = -INFINITY;
    each_group([&](int r, int, const float4& v) {
      mine = fmaxf(mine, near(r, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))));
    });
    float t = reached_by(mine, a.k);
    float floor_ = t - slack(t);
    __syncthreads();
    if (mine > -INFINITY && mine >= floor_) {
      each_group([&](int r, int g0, const float4& v) {
        const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = near(r, w[i]);
          if (u > -INFINITY && u >= floor_) {
            const int to = atomicAdd(&s.n_groups, 1);
            if (to < BP_GROUPS) s.groups[to] = r * a.padded + g0 + i;
          }
        }
      });
    }
    __syncthreads();
    const int ng = s.n_groups;
    if (ng > BP_GROUPS) return false;
    if (!(t > -INFINITY) && ng > BP_LIST / BP_GROUP) {
      // too few threads have groups for a bound: their lanes' best may give one
      mine = -INFINITY;
      for (int j = warp; j < ng; j += BP_THREADS / 32)
        take(j, [&](int r, int, float v) { mine = fmaxf(mine, near(r, v)); });
      t = reached_by(mine, a.k);
      floor_ = t - slack(t);
    }
    for (int j = warp; j < ng; j += BP_THREADS / 32)
      take(j, [&](int r, int v, float x) {
        const float u = near(r, x);
        if (u > -INFINITY && u >= floor_) {
          const int to = atomicAdd(&s.n_list, 1);
          if (to < BP_LIST) {
            s.x[to] = x;
            s.at[to] = (uint32_t)r * a.vocab + v;
          }
        }
      });
    __syncthreads();
    return s.n_list <= BP_LIST;
  }
  template <typename F> RTR_DEVICE void take(int j, F&& f) const {
    const int id = s.groups[j], r = a.n == 1 ? 0 : row_of((uint32_t)id >> 2), g = id - r * a.padded;
    const int first = g * BP_GROUP - Logits<T>::shift(row(r));
    Logits<T> raw;
    raw.load(row(r), first, lane, a.vocab);
    uint32_t bits = 0;
    if constexpr (MASK) bits = allowed_bits<T>(allowed0 + r * a.allowed_stride, first, lane, a.vocab);
    each_logit(r, g, raw, bits, f);
  }

  RTR_DEVICE int block_count(int mine) {
    mine = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) s.red[warp] = mine;
    __syncthreads();
    double all = 0;
    for (int w = 0; w < BP_THREADS / 32; ++w) all += s.red[w];
    return (int)all;
  }

  // The same where ties make the lists too long (rows of equal logits, most of them masked by the type's lowest value): the exact
  // k best groups, by value and place, and of those the exact k best candidates; each by bisection of the
  // value's 64 bits and, among equal ones, of the place.  Rows whose sums differ are summed in 64 bits first.
  template <typename Each> RTR_DEVICE void bisect(Each&& each, int k, uint64_t& least, uint32_t& last) {
    least = 0;  // the largest key that at least k reach (every finite candidate's is above 0)
    for (int b = 63; b >= 0; --b) {
      const uint64_t t = least | 1ull << b;
      int c = 0;
      each([&](uint64_t key, uint32_t) { c += key >= t; });
      if (block_count(c) >= k) least = t;
    }
    int c = 0;
    each([&](uint64_t key, uint32_t) { c += key > least; });
    const int wanted = k - block_count(c);
    last = 0;  // places below it are taken among those of the least key
    if (least == 0) return;
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = last | 1u << b;
      c = 0;
      each([&](uint64_t key, uint32_t at) { c += key == least && at < t; });
      if (block_count(c) <= wanted) last = t;
    }
  }
  __device__ __noinline__ void gather_exactly() {
    for (int r = tid; r < a.n; r += BP_THREADS) {
      bool differs = false;
      for (int q = 0; q < a.n; ++q) differs |= s.off[q] > -INFINITY && s.sum[q] != s.sum[r];
      s.again[r] = differs && s.off[r] > -INFINITY;
    }
    __syncthreads();
    sum_again();
    uint64_t least;
    uint32_t last;
    const auto groups = [&](auto&& f) {
      each_group([&](int r, int g0, const float4& v) {
        const float w[4] = {v.x, v.y, v.z, v.w};
        for (int i = 0; i < 4; ++i)
          if (w[i] > -INFINITY && g0 + i < a.groups) f(double_key(worth(r, w[i])), (uint32_t)(r * a.padded + g0 + i));
      });
    };
    bisect(groups, a.k, least, last);
    if (tid == 0) s.n_groups = s.n_list = 0;
    __syncthreads();
    groups([&](uint64_t key, uint32_t id) {
      if (key > least || (key == least && id < last)) {
        const int to = atomicAdd(&s.n_groups, 1);
        if (to < BP_GROUPS) s.groups[to] = (int32_t)id;
      }
    });
    __syncthreads();
    const int ng = min(s.n_groups, BP_GROUPS);
    const auto logits = [&](auto&& f) {
      for (int j = warp; j < ng; j += BP_THREADS / 32)
        take(j, [&](int r, int v, float x) { f(double_key(worth(r, x)), (uint32_t)r * a.vocab + v, x); });
    };
    bisect([&](auto&& f) { logits([&](uint64_t key, uint32_t at, float) { f(key, at); }); }, a.k, least, last);
    logits([&](uint64_t key, uint32_t at, float x) {
      if (key > least || (key == least && at < last)) {
        const int to = atomicAdd(&s.n_list, 1);
        if (to < BP_LIST) {
          s.x[to] = x;
          s.at[to] = at;
        }
      }
    });
    __syncthreads();
  }

  // Candidates by value, then place: each one's rank is the number of those before it.
  RTR_DEVICE void put_in_order() {
    const int n = s.n_list;
    for (int i = tid; i < n; i += BP_THREADS) s.key[i] = double_key(worth(s.at[i] / a.vocab, s.x[i]));
    __syncthreads();
    for (int i = warp; i < n; i += BP_THREADS / 32) {
      const uint64_t key = s.key[i];
      const uint32_t at = s.at[i];
      int before = 0;
      for (int j = lane; j < n; j += 32) before += s.key[j] > key || (s.key[j] == key && s.at[j] < at);
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) s.order[before] = (uint16_t)i;
    }
    __syncthreads();
  }

  // Marks the rows of candidates among (or just behind) the first k that are too close to those of another row.  Rows whose
  // sums are equal have exact differences, as long as either all of them are summed again or none.
  RTR_DEVICE bool doubtful() {
    if (tid == 0) s.doubts = 0;
    __syncthreads();
    const int n = s.n_list;
    for (int i = tid; i + 1 < n; i += BP_THREADS) {
      // behind the k-th everything is compared with that one
      const int p = s.order[min(i, a.k - 1)], q = s.order[i + 1];
      const int rp = s.at[p] / a.vocab, rq = s.at[q] / a.vocab;
      if (rp == rq || s.sum[rp] == s.sum[rq] || (s.done[rp] && s.done[rq])) continue;
      if (key_double(s.key[p]) - key_double(s.key[q]) >= BP_DOUBT) continue;
      s.again[rp] = s.again[rq] = 1;
      s.doubts = 1;
    }
    __syncthreads();
    if (!s.doubts) return false;
    bool equal = false;
    if (tid < a.n && s.off[tid] > -INFINITY)
      for (int q = 0; q < a.n; ++q) equal |= s.again[q] && s.sum[q] == s.sum[tid];
    __syncthreads();
    if (equal) s.again[tid] = 1;
    __syncthreads();
    return true;
  }
};

template <typename T, bool MASK>
__global__ void __launch_bounds__(BP_THREADS) beam_pick_kernel(const BeamPick a) {
  __shared__ PickShared s;
  pdl_launch_dependents();
  pdl_wait();
  const int item = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row0 = (int64_t)item * a.n;
  Picker<T, MASK> p{a, s, item, tid, warp, lane, static_cast<const T*>(a.logits) + row0 * a.stride,
                    MASK ? a.allowed + row0 * a.allowed_stride : nullptr, a.best + row0 * a.padded};
  p.offsets();
  if (!p.gather()) p.gather_exactly();
  p.put_in_order();
  if (p.doubtful()) {
    p.sum_again();
    p.put_in_order();
  }
  // fewer finite candidates than k: the first places that have none
  const int n = min(s.n_list, a.k);
  if (n < a.k) {
    const int64_t all = (int64_t)a.n * a.vocab;
    bool free_ = tid < 2 * a.k && tid < all;
    for (int j = 0; j < n && free_; ++j) free_ = s.at[j] != (uint32_t)tid;
    const unsigned mask = __ballot_sync(0xffffffffu, free_);
    if (lane == 0) s.red[warp] = __popc(mask);
    __syncthreads();
    int before = __popc(mask & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) before += (int)s.red[w];
    if (free_ && n + before < a.k) {
      s.at[n + before] = (uint32_t)tid;
      s.key[n + before] = double_key(-INFINITY);
      s.order[n + before] = (uint16_t)(n + before);
    }
    __syncthreads();
  }
  if (tid < a.k) {
    const int i = s.order[tid];
    const int64_t to = (int64_t)item * a.k + tid;
    a.all_tokens[to] = s.at[i] % a.vocab;
    a.all_parents[to] = s.at[i] / a.vocab;
    a.all_scores[to] = (float)key_double(s.key[i]);
  }
  if (warp == 0) {
    int taken = 0;
    for (int j0 = 0; j0 < a.k && taken < a.beams; j0 += 32) {
      const int j = j0 + lane;
      const int i = j < a.k ? s.order[j] : 0, token = s.at[i] % a.vocab;
      const bool on = j < a.k && token != a.eos;
      const unsigned mask = __ballot_sync(0xffffffffu, on);
      const int place = taken + __popc(mask & ((1u << lane) - 1));
      if (on && place < a.beams) {
        const int64_t to = (int64_t)item * a.beams + place;
        a.next_tokens[to] = token;
        a.next_parents[to] = s.at[i] / a.vocab;
        a.next_scores[to] = (float)key_double(s.key[i]);
      }
      taken += __popc(mask);
    }
  }
}

// --------------------------------------------------------------------- host
static const char* beam_check(const rtr_beam_step* b) {
  if (!b) return "null step";
  if (b->dtype != RTR_DTYPE_F32 && b->dtype != RTR_DTYPE_BF16) return "dtype must be float32 or bfloat16";
  if (b->items < 0 || b->n < 1 || b->n > BP_MAX_N) return "1 to 128 beams an item";
  if (b->vocab < 1 || b->vocab > 1 << 20) return "a vocabulary of 1 to 2^20 tokens";
  if (b->k < 1 || b->k > BP_MAX_K || b->k > (int64_t)b->n * b->vocab) return "1 to 256 candidates, and no more than there are";
  if (b->beams < 1 || b->beams > b->k) return "the next beams must be some of the candidates";
  if (b->eos >= 0 && b->k < b->beams + b->n) return "with eos the candidates must be at least the next beams and the former ones";
  if (b->items > 1 || b->n > 1)
    if (b->logits_stride < b->vocab) return "rows of logits overlap";
  if (b->allowed && b->allowed_stride != 0 && b->allowed_stride < b->vocab) return "rows of allowed overlap";
  if (b->items && (!b->logits || !b->scores || !b->all_tokens || !b->all_parents || !b->all_scores || !b->next_tokens ||
                   !b->next_parents || !b->next_scores || !b->status))
    return "null buffer";
  if (reinterpret_cast<uintptr_t>(b->logits) % (b->dtype == RTR_DTYPE_F32 ? 4 : 2)) return "logits must lie at multiples of their size";
  return nullptr;
}

// Groups of a row (one more where it starts in the middle of one), slices, and the workspace they need.
static void beam_plan(const rtr_beam_step* b, int sms, BeamPick& p, int64_t& best_bytes, int64_t& bytes) {
  const int per = b->dtype == RTR_DTYPE_F32 ? 4 : 8;
  p.groups = (int)(((int64_t)b->vocab + per - 1 + BP_GROUP - 1) / BP_GROUP);
  p.padded = (p.groups + 3) & ~3;
  p.quarter_inv = (uint32_t)((0x100000000ull + p.padded / 4 - 1) / (p.padded / 4));
  // A slice is two rounds of a block's warps where the rows alone fill the GPU, and one where they do not
  const int64_t rows = (int64_t)b->items * b->n;
  const int round = BP_WARPS * BP_AHEAD;
  int64_t slices = (p.groups + 2 * round - 1) / (2 * round);
  if (rows * slices < 4 * (int64_t)sms) slices = (p.groups + round - 1) / round;
  p.slices = (int)slices;
  best_bytes = rows * p.padded * (int64_t)sizeof(float);
  best_bytes = (best_bytes + 15) & ~(int64_t)15;
  bytes = best_bytes + rows * p.slices * (int64_t)sizeof(float2);
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_beam_select_workspace(const rtr_beam_step* step, int32_t device, int64_t* bytes) {
  if (const char* e = beam_check(step)) return set_error(RTR_ERR_ARG, e);
  if (!bytes) return set_error(RTR_ERR_ARG, "null size");
  cudaError_t e = cudaSuccess;
  const int sms = kv_sms(device, e);
  if (e != cudaSuccess) return set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
  BeamPick p;
  int64_t best;
  beam_plan(step, sms, p, best, *bytes);
  return RTR_OK;
}

int rtr_beam_select(const rtr_beam_step* step, void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
  if (const char* e = beam_check(step)) return set_error(RTR_ERR_ARG, e);
  if (!step->items) return RTR_OK;
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  BeamPick p = {};
  int64_t best = 0, bytes = 0;
  beam_plan(step, on.sms, p, best, bytes);
  if (!workspace || workspace_bytes < bytes || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(RTR_ERR_ARG, "the workspace is too small or not aligned to 16 bytes");
  const int64_t blocks = (int64_t)step->items * step->n * p.slices;
  if (blocks > INT32_MAX) return set_error(RTR_ERR_ARG, "too many rows for one call");
  p.logits = step->logits;
  p.scores = step->scores;
  p.allowed = step->allowed;
  p.stride = step->logits_stride;
  p.allowed_stride = step->allowed_stride;
  p.items = step->items;
  p.n = step->n;
  p.vocab = step->vocab;
  p.k = step->k;
  p.beams = step->beams;
  p.eos = step->eos < 0 ? -1 : step->eos;
  p.best = static_cast<float*>(workspace);
  p.part = reinterpret_cast<float2*>(static_cast<char*>(workspace) + best);
  p.all_tokens = step->all_tokens;
  p.all_parents = step->all_parents;
  p.all_scores = step->all_scores;
  p.next_tokens = step->next_tokens;
  p.next_parents = step->next_parents;
  p.next_scores = step->next_scores;
  p.status = step->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto run = [&](auto scan, auto pick) {
    const cudaError_t e = kv_launch(scan, dim3((unsigned)blocks), BP_WARPS * 32, 0, 1, st, p);
    return e == cudaSuccess ? kv_launch(pick, dim3((unsigned)p.items), BP_THREADS, 0, 1, st, p) : e;
  };
  cudaError_t e;
  if (step->dtype == RTR_DTYPE_F32)
    e = p.allowed ? run(beam_scan_kernel<float, true>, beam_pick_kernel<float, true>)
                  : run(beam_scan_kernel<float, false>, beam_pick_kernel<float, false>);
  else
    e = p.allowed ? run(beam_scan_kernel<__nv_bfloat16, true>, beam_pick_kernel<__nv_bfloat16, true>)
                  : run(beam_scan_kernel<__nv_bfloat16, false>, beam_pick_kernel<__nv_bfloat16, false>);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
