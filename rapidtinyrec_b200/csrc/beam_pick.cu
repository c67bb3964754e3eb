// The best continuations of beams over the whole vocabulary, from one pass over the logits.
//
// Mathematics.  Candidate (i, v) is worth x[i][v] - lse[i] + score[i] with lse the log of the sum
// of exponentials of row i.  Within a row the order is that of the logits; across rows it needs lse, which is known
// only when a row has been read.  So the first kernel reads each logit once and leaves, beside each slice's
// maximum and sum, of every group of 2 KB of logits the largest (of those that are allowed), which lane of the
// warp had it, and the largest of the other lanes.  The k-th largest of the groups' best is a lower bound of the k-th largest
// candidate, and only groups whose best reaches it can hold one of the k: k of them but for ties.  The second kernel (a
// block an item) finds a bound just below that one, by counting how far its threads' groups lie behind the best; takes the
// groups that reach it and of each the 32 or 64 bytes of the lane that has it (all lanes where another one may
// have more); and puts what reaches the bound in order: for 100 candidates of 50 beams some 7 KB of
// 30 MB are read again.
//
// Order.  Sums are fp32, their logs off by some 1e-6 at most (beam_close has the bound; in 27,648 rows of 1,000 to 2^20 logits, normal ones,
// ramps and rows of one or two values among them, by -5.2e-7 to 3.1e-7).  The 100 best of
// 7.6 million candidates lie 1e-4 to 1e-3 apart, so now and then two are too close to tell.  Differences of logits and scores are exact
// enough in fp64; what is not known well is the sum.  Where two neighbours of different rows are closer than BeamPick::close, twice that
// bound, both rows' sums are taken again in fp64 (rows whose fp32 sums are the same among them) and the list is put in order
// again (two rows of 152,832: 63 us more by one block, some 25 by the four that are there in a batch; for one item in 80 or so): the
// order is that of 64-bit arithmetic, however the rows were split.
// What bounds it.  The first kernel: exponentials (XU 80 %) and issue slots (62 %), 1,600 rows of 152,832 in bf16 in 82 us, 5.96 TB/s;
// without its exponentials it reads at 7.3 TB/s.  An eighth or a quarter of them on the FMA pipe instead: no change, and 3 us slower.
// The second: latency, some 17,800 cycles, 9 us, for 50 beams: dependent loads (slices and groups, second bests, lanes' logits; 700
// to 2,500 cycles each), code that comes from L2 as it is gone through once, and a dozen barriers of 1,024 threads (512 threads: 0.4 us
// less for 4 beams, 0.9 more for 50).
//
// What the usual path is not made for: one beam far ahead of the others, masks that leave few groups (gather_closely, 25 to 50 us), and
// ties that make its lists too long (gather_exactly: 0.4 ms for 4 rows of 8,192 equal logits, 1.8 ms for 50 of 152,832).
#include <cuda_runtime.h>

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "engine.h"
#include "kv_attention.cuh"
#include "kv_host.h"

namespace rtr {

constexpr int BP_BYTES = 2048;                  // of a group: four pieces of 16 of each lane of a warp
constexpr int BP_WARPS = 8;                     // first kernel: warps of a block
constexpr int beam_blocks(bool mask) { return mask ? 3 : 4; }  // blocks of an SM
constexpr int BP_RING = 6144;                   // bytes of logits that a warp of it has on their way
constexpr int BP_THREADS = 1024;                // second kernel: threads of a block
constexpr int BP_MAX_N = 128, BP_MAX_K = 256;
constexpr int BP_GROUPS = 512, BP_LANES = 1024, BP_LIST = 1024;  // groups, lanes of them and candidates that it takes up at once
constexpr int BP_HELD = 4;                      // quartets of groups that a thread of it holds
constexpr int BP_RANKS = 4;                     // blocks that sum an item's doubtful rows together
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
  float close;             // see beam_close
  int ranks;               // blocks of the second kernel's clusters
  float* best;             // [items * n][padded]: a group's largest allowed logit
  uint32_t* second;        // likewise: the largest of the other lanes' (rounded up) and, in the last five bits, whose the first is
  float2* part;            // [items * n][slices]: maximum, sum of exponentials relative to 2^beam_unit of it, or to it
  int32_t *all_tokens, *all_parents, *next_tokens, *next_parents;
  float *all_scores, *next_scores;
  uint32_t* status;
};

RTR_DEVICE float redux_max(float v) {  // NaN counts as nothing
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// What a sum of exponentials with the largest logit `base` is relative to, as a power of two.  Where base is within 2^21 that is
// the whole number nearest to base log2(e), less 8: exponents are x log2(e) less it, rounded once as what is left (which is least
// about 0, so that is put where the many are and not at the best), and sums change from one to another by exact powers of two.
// Beyond (all of a slice masked by -1e10, say) the rounding of base log2(e) itself would be what is left, so there the difference x - base
// comes first, which is exact wherever it counts: such logits are a quarter apart at least.
constexpr float BP_NEAR = 0x1p21f;
RTR_DEVICE bool beam_near(float base) { return fabsf(base) < BP_NEAR; }
RTR_DEVICE float beam_unit(float base) {
  const float whole = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers
  return __fadd_rn(__fmaf_rn(fmaxf(base, -BP_NEAR), BP_LOG2E, whole), -whole - 8.f);
}
RTR_DEVICE double beam_offset(float base) { return beam_near(base) ? beam_unit(base) - (double)base * BP_LOG2E : 0.0; }
// A sum of `base` times this is one of `top`, another and larger base: of two that are near (a base below -2^21 as if it were that),
// and of any.
RTR_DEVICE float beam_power(float d) { return d < -126.f ? 0.f : __int_as_float((127 + (int)d) << 23); }  // 2^d, d a whole number
RTR_DEVICE float beam_near_scale(float base, float top) { return beam_power(beam_unit(base) - beam_unit(top)); }
__device__ __noinline__ float beam_far_scale(float base, float top) {
  return (float)exp2(((double)base - top) * 1.4426950408889634 + beam_offset(base) - beam_offset(top));
}
RTR_DEVICE float beam_relative(const float2& part, float top) {  // part: a base and its sum
  if (part.x == top || part.y == 0.f) return part.y;
  return part.y * (beam_near(part.x) && beam_near(top) ? beam_near_scale(part.x, top) : beam_far_scale(part.x, top));
}
struct BeamSum {
  double sum;
  float base;
};
RTR_DEVICE double beam_warp_sum(double v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A piece of 16 bytes at a row's ragged ends, of which some logits are not there.  Out of line: the code that a
// kernel goes through once comes from L2 at some 500 cycles a line.
template <typename T> __device__ __noinline__ uint4 beam_ragged(const T* row, int e, int vocab) {
  constexpr int PER = 16 / sizeof(T);
  uint32_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = sizeof(T) == 4 ? 0xff800000u : 0xff80u;
    if (e + i >= 0 && e + i < vocab) {
      if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(row[e + i]);
      else v[i] = __bfloat16_as_ushort(row[e + i]);
    }
  }
  if constexpr (sizeof(T) == 4) return make_uint4(v[0], v[1], v[2], v[3]);
  else return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// A warp's part of a group (1,024 logits in bf16, 512 in fp32), four pieces of 16 bytes each lane.  Groups start at multiples
// of 16 bytes: the first of a row that does not holds fewer.
template <typename T> struct Logits {
  static constexpr int PER = 16 / sizeof(T), PIECES = 4, EACH = PIECES * PER, GROUP = 32 * EACH;
  uint4 u[PIECES];
  RTR_DEVICE static int shift(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
  RTR_DEVICE static int at(int first, int i, int lane) { return first + (i / PER) * 32 * PER + lane * PER + i % PER; }
  RTR_DEVICE void none() {
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) u[j] = make_uint4(w, w, w, w);
  }
  RTR_DEVICE void load_inside(const T* p) {  // p: the lane's first logit of a group that is all there
#pragma unroll
    for (int j = 0; j < PIECES; ++j) u[j] = __ldg(reinterpret_cast<const uint4*>(p + j * 32 * PER));
  }
  RTR_DEVICE void load(const T* row, int first, int lane, int vocab) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int e = at(first, j * PER, lane);
      if (e >= 0 && e + PER <= vocab) {
        u[j] = __ldg(reinterpret_cast<const uint4*>(row + e));
      } else {
        u[j] = beam_ragged(row, e, vocab);
      }
    }
  }
  RTR_DEVICE float2 two(int i) const {  // logits 2 i and 2 i + 1
    const uint4& p = u[i / (PER / 2)];
    if constexpr (sizeof(T) == 4) {
      return i & 1 ? make_float2(__uint_as_float(p.z), __uint_as_float(p.w)) : make_float2(__uint_as_float(p.x), __uint_as_float(p.y));
    } else {
      const uint32_t w = (i & 3) == 0 ? p.x : (i & 3) == 1 ? p.y : (i & 3) == 2 ? p.z : p.w;
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
  }
  RTR_DEVICE float one(int i) const { return i & 1 ? two(i >> 1).y : two(i >> 1).x; }
  RTR_DEVICE float largest() const {
    if constexpr (sizeof(T) == 4) {
      float m[PIECES];
#pragma unroll
      for (int j = 0; j < PIECES; ++j) m[j] = fmaxf(fmaxf(one(4 * j), one(4 * j + 1)), fmaxf(one(4 * j + 2), one(4 * j + 3)));
      return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    } else {  // two at a time; NaN counts as nothing
      const auto pair = [](uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); };
      const auto four = [&](const uint4& x) { return __hmax2(__hmax2(pair(x.x), pair(x.y)), __hmax2(pair(x.z), pair(x.w))); };
      const __nv_bfloat162 m = __hmax2(__hmax2(four(u[0]), four(u[1])), __hmax2(four(u[2]), four(u[3])));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};
// The word of BeamPick::second, and the value that its largest is at most.
RTR_DEVICE uint32_t beam_second(float value, int lane) { return (__float_as_uint(value) & ~31u) | (uint32_t)lane; }
RTR_DEVICE float beam_second_value(uint32_t w) { return __uint_as_float(w >> 31 ? w & ~31u : w | 31u); }

// The bytes that say which of a lane's logits are allowed: runs of four, by aligned words that hold at least one
// of them, since a row of bytes may start anywhere (at the same place of a word in all of a row's groups).
template <typename T> struct Allowed {
  static constexpr int RUNS = Logits<T>::EACH / 4;
  uint32_t w[RUNS][2];
  RTR_DEVICE static int by(const uint8_t* row, int shift) { return 8 * (int)((reinterpret_cast<uintptr_t>(row) - shift) & 3); }
  RTR_DEVICE void load_inside(const uint8_t* row, int first, int lane, int by) {  // a group that is all there
    if (Logits<T>::PER == 8 && (reinterpret_cast<uintptr_t>(row + first) & 7) == 0) {
#pragma unroll
      for (int j = 0; j < RUNS; j += 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + Logits<T>::at(first, 4 * j, lane)));
        w[j][0] = u.x;
        w[(j + 1) % RUNS][0] = u.y;
      }
      return;
    }
    const uintptr_t p = reinterpret_cast<uintptr_t>(row + Logits<T>::at(first, 0, lane)) & ~(uintptr_t)3;
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p + (Logits<T>::at(0, 4 * j, lane) - Logits<T>::at(0, 0, lane)));
      w[j][0] = __ldg(q);
      if (by) w[j][1] = __ldg(q + 1);
    }
  }
  RTR_DEVICE void load(const uint8_t* row, int first, int lane, int vocab, int by) {
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
      const int e = Logits<T>::at(first, 4 * j, lane);
      w[j][0] = w[j][1] = 0;
      if (e >= 0 && e + 4 <= vocab) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(row + e) & ~(uintptr_t)3);
        w[j][0] = __ldg(p);
        if (by) w[j][1] = __ldg(p + 1);
      } else {  // a row's ragged ends
        uint64_t four = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e + i >= 0 && e + i < vocab) four |= (uint64_t)row[e + i] << (8 * i);
        four <<= by;
        w[j][0] = (uint32_t)four;
        w[j][1] = (uint32_t)(four >> 32);
      }
    }
  }
  RTR_DEVICE bool operator()(int i, int by) const {
    return __funnelshift_r(w[i >> 2][0], w[i >> 2][1], by) >> (8 * (i & 3)) & 0xffu;
  }
  // The largest allowed one of the lane's logits: the others become NaN, which counts as nothing.
  RTR_DEVICE float largest(const Logits<T>& raw, int by) const {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
      const uint32_t none = __vcmpeq4(__funnelshift_r(w[j][0], w[j][1], by), 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m = fmaxf(m, __uint_as_float(__float_as_uint(raw.one(4 * j + i)) | __byte_perm(none, 0u, 0x1111 * i)));
    }
    return m;
  }
};

// The sum of the exponentials of a warp's groups relative to m, the slice's largest logit, where that is beyond 2^21: exponents are
// rounded about 8 as above.  (50 rows of 152,704 of which all but 1,000 are masked by -1e10: 46 us, by -1e4 42, by minus
// infinity 22; with exponentials in 64 bits 57.)
template <typename T> __device__ __noinline__ double beam_far_sum(const T* row, float m, int g, int hi, int vocab) {
  using L = Logits<T>;
  const int lane = threadIdx.x & 31, shift = L::shift(row);
  const float2 less = make_float2(-m, -m), log2e = make_float2(BP_LOG2E, BP_LOG2E), eight = make_float2(8.f, 8.f);
  double sum = 0.0;
  L next;
  if (g < hi) next.load(row, g * L::GROUP - shift, lane, vocab);
  for (; g < hi; g += BP_WARPS) {
    const L raw = next;
    if (g + BP_WARPS < hi) next.load(row, (g + BP_WARPS) * L::GROUP - shift, lane, vocab);
    float2 part[4];
#pragma unroll
    for (int i = 0; i < L::EACH / 2; ++i) {
      const float2 y = __ffma2_rn(__fadd2_rn(raw.two(i), less), log2e, eight), e = make_float2(ex2(y.x), ex2(y.y));
      part[i & 3] = i < 4 ? e : __fadd2_rn(part[i & 3], e);
    }
    const float2 more = __fadd2_rn(__fadd2_rn(part[0], part[1]), __fadd2_rn(part[2], part[3]));
    sum += (double)more.x + more.y;
  }
  return beam_warp_sum(sum) * 0x1p-8;
}

// One block: a slice of a row's groups, which its warps take in turn.  The groups that are all there come through a ring in shared
// memory of each warp's own, every lane's pieces copied by the lane that reads them: 6 KB a warp keep 192 KB an SM on their way without
// a register (two groups in registers, one read while the other comes, 24 warps an SM: 110 us instead of 96 for 32 x 50 rows of bf16 and
// the second kernel as it was then).
template <typename T, bool MASK>
__global__ void __launch_bounds__(BP_WARPS * 32, beam_blocks(MASK)) beam_scan_kernel(const BeamPick a) {
  using L = Logits<T>;
  constexpr int BYTES = BP_BYTES, STAGES = BP_RING / BYTES, GROUP = L::GROUP;
  __shared__ __align__(16) uint8_t ring[BP_WARPS][BP_RING];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const float score = a.scores[row];
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const uint8_t* allowed = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  const int shift = L::shift(x), by = MASK ? Allowed<T>::by(allowed, shift) : 0;
  const int lo = (int)((int64_t)a.groups * slice / a.slices), hi = (int)((int64_t)a.groups * (slice + 1) / a.slices);
  float* best = a.best + (int64_t)row * a.padded;
  if (!(score > -INFINITY)) {  // minus infinity: nothing to offer; NaN: the second kernel reports it
    if (tid == 0) a.part[blockIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  if (slice == a.slices - 1 && tid < a.padded - a.groups) best[a.groups + tid] = -INFINITY;
  float base = -INFINITY, unit = beam_unit(base);
  // A group's exponentials are added to one another, and that to the running sum; what these additions lose is a sum of its
  // own (all in one running sum: rows of 152,832 of one value off by up to 1.3e-6; no faster).
  float2 sum = make_float2(0.f, 0.f), lost = sum;
  const float2 log2e = make_float2(BP_LOG2E, BP_LOG2E);
  const auto take = [&](const L& raw, const Allowed<T>& ok, int g) {
    float mine = raw.largest();
    const float top = redux_max(mine);
    float most = top;
    if constexpr (MASK) {
      mine = ok.largest(raw, by);
      most = redux_max(mine);
    }
    const int whose = __ffs(__ballot_sync(0xffffffffu, mine == most)) - 1;
    const float other = redux_max(lane == whose ? -INFINITY : mine);
    if (lane == 0) {
      best[g] = most;
      a.second[(int64_t)row * a.padded + g] = beam_second(other, whose & 31);
    }
    if (top > base) {  // the same in all lanes.  (Beyond 2^21 what is summed means nothing: see the end.)
      base = top;
      const float to = beam_unit(base), f = beam_power(unit - to);
      unit = to;
      sum = make_float2(sum.x * f, sum.y * f);
      lost = make_float2(lost.x * f, lost.y * f);
    }
    const float2 minus = make_float2(-unit, -unit), less = make_float2(-1.f, -1.f);
    float2 part[4];
#pragma unroll
    for (int i = 0; i < L::EACH / 2; ++i) {
      const float2 y = __ffma2_rn(raw.two(i), log2e, minus), e = make_float2(ex2(y.x), ex2(y.y));
      part[i & 3] = i < 4 ? e : __fadd2_rn(part[i & 3], e);
    }
    const float2 more = __fadd2_rn(__fadd2_rn(part[0], part[1]), __fadd2_rn(part[2], part[3])), now = __fadd2_rn(sum, more);
    lost = __fadd2_rn(lost, __ffma2_rn(__ffma2_rn(sum, less, now), less, more));
    sum = now;
  };
  // the warp's groups that are all there, and before and behind them those at the row's ends
  const int end = min(hi, (int)(((int64_t)a.vocab + shift) / GROUP));
  int g = lo + warp;
  L raw;
  Allowed<T> ok;
  if (g == 0 && shift && hi > 0) {
    raw.load(x, -shift, lane, a.vocab);
    if constexpr (MASK) ok.load(allowed, -shift, lane, a.vocab, by);
    take(raw, ok, 0);
    g = BP_WARPS;
  }
  const int n = g < end ? (end - g + BP_WARPS - 1) / BP_WARPS : 0;
  const T* from = x + ((int64_t)g * GROUP - shift + lane * L::PER);
  uint8_t* mine = ring[warp] + lane * 16;
  const auto issue = [&](int i, int stage) {
    if (i < n) {
#pragma unroll
      for (int j = 0; j < L::PIECES; ++j)
        cp_async16(mine + stage * BYTES + j * 512, from + (int64_t)i * (BP_WARPS * GROUP) + j * 32 * L::PER, true);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i, i);
  Allowed<T> next;  // masks come a group ahead, in registers
  if constexpr (MASK)
    if (n > 0) next.load_inside(allowed, g * GROUP - shift, lane, by);
  for (int i = 0, stage = 0; i < n; ++i) {
    if constexpr (MASK) {
      ok = next;
      if (i + 1 < n) next.load_inside(allowed, (g + (i + 1) * BP_WARPS) * GROUP - shift, lane, by);
    }
    cp_async_wait<STAGES - 2>();
    __syncwarp();
#pragma unroll
    for (int j = 0; j < L::PIECES; ++j) raw.u[j] = *reinterpret_cast<const uint4*>(mine + stage * BYTES + j * 512);
    __syncwarp();
    issue(i + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);  // where the last one was
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    take(raw, ok, g + i * BP_WARPS);
  }
  for (g += n * BP_WARPS; g < hi; g += BP_WARPS) {
    raw.load(x, g * GROUP - shift, lane, a.vocab);
    if constexpr (MASK) ok.load(allowed, g * GROUP - shift, lane, a.vocab, by);
    take(raw, ok, g);
  }
  const double total = beam_warp_sum(((double)sum.x + sum.y) + ((double)lost.x + lost.y));
  const auto sums = [&](int w) -> BeamSum& { return *reinterpret_cast<BeamSum*>(ring[w]); };  // nothing is under way any more
  if (lane == 0) sums(warp) = BeamSum{total, base};
  __syncthreads();
  // a slice whose largest logit is beyond 2^21 is read once more
  const float m = redux_max(lane < BP_WARPS ? sums(lane).base : -INFINITY);
  if (!beam_near(m) && m > -INFINITY) {
    __syncthreads();
    const double far = beam_far_sum(x, m, lo + warp, hi, a.vocab);
    if (lane == 0) sums(warp) = BeamSum{far, m};
    __syncthreads();
  }
  if (warp == 0) {
    const BeamSum u = lane < BP_WARPS ? sums(lane) : BeamSum{0.0, -INFINITY};
    double t = u.base == m ? u.sum : u.sum * beam_near_scale(u.base, m);
#pragma unroll
    for (int d = BP_WARPS / 2; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (lane == 0) a.part[blockIdx.x] = make_float2(m, (float)t);
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

// e^d for d from -100 to 0: e^(n log 2 + f) with n the nearest whole number, f at most 0.347 and e^f its Taylor series up to f^10 / 10!
// (off by 2.2e-13 at most).  Sixteen fp64 operations with the subtraction and the sum; exp() made two rows of 152,704 take 95 us.
RTR_DEVICE double exp_of(double d) {
  const double whole = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to whole numbers, in the low bits
  const double z = fma(d, 1.4426950408889634, whole), n = z - whole, f = fma(n, -0.69314718055994531, d);
  double e = 1.0 / 3628800.0;
  e = fma(e, f, 1.0 / 362880.0);
  e = fma(e, f, 1.0 / 40320.0);
  e = fma(e, f, 1.0 / 5040.0);
  e = fma(e, f, 1.0 / 720.0);
  e = fma(e, f, 1.0 / 120.0);
  e = fma(e, f, 1.0 / 24.0);
  e = fma(e, f, 1.0 / 6.0);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.0);
  e = fma(e, f, 1.0);
  return __hiloint2double(__double2hiint(e) + (__double2loint(z) << 20), __double2loint(e));
}

struct PickEntry {  // a candidate in order: larger keys first, then lower places
  uint64_t key;
  uint32_t at, row;
};
struct PickShared {
  double sum[BP_MAX_N], off[BP_MAX_N];  // log of the sum of exponentials relative to the maximum, score - that
  float2 near[BP_MAX_N];                // the row's maximum, and off rounded (minus infinity: nothing to offer)
  float need[BP_MAX_N];                 // what its logits have to reach
  uint8_t again[BP_MAX_N], done[BP_MAX_N];  // rows to sum in 64 bits, and those that are
  double share[BP_RANKS][BP_MAX_N];         // and what the blocks of the cluster have of their sums
  int doubt;                                // whether there are any
  int32_t quartet_at[BP_GROUPS], groups[BP_GROUPS];
  PickEntry list[BP_LIST];
  uint16_t order[BP_LIST];              // and their places in the list
  union {
    int bins[BP_THREADS];               // of the search for the k-th best
    float x[BP_LIST];                   // and then the candidates' logits
  };
  double red[BP_THREADS / 32];
  union {
    float4 quartet[BP_GROUPS];          // quartets of groups one of which reaches the row's need
    int2 lane[BP_LANES];                // and then the lanes whose largest logit does: 32 row + lane, first place of the group
  };
  int n_quartets, n_groups, n_whole, n_lanes, n_list;
  int word2[BP_THREADS / 32];
  uint32_t word[BP_THREADS / 32], reached, above;
  int most;  // the largest |off32|, as bits
  int wild;  // whether a row's largest logit or its offset is above 1e30
};

// A count in shared memory that other threads are adding to.
RTR_DEVICE int so_far(const int& count) { return *const_cast<const volatile int*>(&count); }

// A value that at least k of many reach, and few more, or minus infinity where fewer are finite; each(f) calls f with a thread's
// values.  They are counted by how far their keys lie behind the largest, in bins of 1/32 of that distance: one pass
// and one scan (with one value a thread 1,200 cycles; finding the value bit by bit, with a barrier each, 2,600).  FINER: by how far they
// lie behind s.above, which a call leaves where its bin ends above.  MANY: values may be the same, and a bin that has k counts no more.
template <bool FINER, bool MANY = true, typename Each> RTR_DEVICE float reached_among(Each&& each, int k, PickShared& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const auto key_of = [](float v) { return v > -INFINITY ? float_key(v) : 0u; };
  uint32_t key = 0;
  if constexpr (!FINER) each([&](float v) { key = max(key, key_of(v)); });
  const uint32_t warp_most = __reduce_max_sync(0xffffffffu, key);
  s.bins[tid] = 0;
  if (lane == 0) s.word[warp] = warp_most;
  __syncthreads();
  const uint32_t most = FINER ? s.above : __reduce_max_sync(0xffffffffu, s.word[lane]);
  each([&](float v) {
    const uint32_t u = key_of(v), bits = __float_as_uint((float)(most - min(u, most)));
    int* bin = &s.bins[bits ? min(BP_THREADS - 1, (int)(bits >> 18) - (127 << 5) + 1) : 0];
    if (u && (!MANY || so_far(*bin) < k)) atomicAdd(bin, 1);
  });
  __syncthreads();
  const int c = s.bins[tid];
  int sum = c;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += u;
  }
  if (lane == 31) s.word2[warp] = sum;
  if (tid == 0) s.reached = 0;
  __syncthreads();
  int before = lane < warp ? s.word2[lane] : 0;
  sum += __reduce_add_sync(0xffffffffu, before);
  // the last bin holds whatever is further away than it starts: no bound
  if (tid < BP_THREADS - 1 && sum >= k && sum - c < k) {
    const auto behind = [&](int bin) {  // the key where a bin starts
      return most - min(most, bin > 0 ? (uint32_t)ceilf(__uint_as_float((uint32_t)(bin - 1 + (127 << 5)) << 18)) : 0u);
    };
    s.reached = max(0x00800000u, tid ? behind(tid + 1) : most);  // no further than the least float
    s.above = behind(tid);
  }
  __syncthreads();
  return s.reached ? key_float(s.reached) : -INFINITY;
}
// The same of one value a thread.
RTR_DEVICE float reached_by(float mine, int k, PickShared& s) {
  return reached_among<false, false>([&](auto&& f) { f(mine); }, k, s);
}
// What the usual path does not come by, out of line.
template <typename T, bool MASK> __device__ __noinline__ void pick_closely(const BeamPick& a, PickShared& s);
template <typename T, bool MASK> __device__ __noinline__ void pick_exactly(const BeamPick& a, PickShared& s);
template <typename T, bool MASK> __device__ __noinline__ void pick_needs(const BeamPick& a, PickShared& s, int ng);
template <typename T, bool MASK> __device__ __noinline__ void pick_whole(const BeamPick& a, PickShared& s);
template <typename T, bool MASK> __device__ __noinline__ void pick_again(const BeamPick& a, PickShared& s);
__device__ __noinline__ void pick_fill(const BeamPick& a, PickShared& s);

template <typename T, bool MASK> struct Picker {
  using L = Logits<T>;
  const BeamPick& a;
  PickShared& s;
  const int item, tid, warp, lane;
  const T* x0;               // the item's first row
  const uint8_t* allowed0;
  const float* best;         // [n][padded]

  RTR_DEVICE int row_of(uint32_t quartet) const { return (int)(a.quarter_inv ? __umulhi(quartet, a.quarter_inv) : quartet); }
  RTR_DEVICE const T* row(int r) const { return x0 + r * a.stride; }
  // what a candidate is worth, and nearly so
  RTR_DEVICE double worth(int r, float x) const { return ((double)x - (double)s.near[r].x) + s.off[r]; }
  RTR_DEVICE float near(int r, float x) const { return (x - s.near[r].x) + s.near[r].y; }
  RTR_DEVICE bool alive(int r) const { return s.near[r].y > -INFINITY; }
  // A value below float32's range, which rounds to minus infinity, counts as that.  Where none of an item's rows reaches 1e30 by a
  // logit or its offset, those are the ones that `near` has as minus infinity.
  RTR_DEVICE static bool counts(double value) { return value > -0x1.ffffffp127; }

  // The thread's quartets of groups: the first ones are held in registers, from the start of the kernel.  Where there is not one for
  // every thread, groups are dealt one by one, as quartets whose others are minus infinity: the fewer a thread has, the nearer
  // to the k-th best candidate is the k-th best thread's.
  float4 held[BP_HELD];
  RTR_DEVICE bool single() const { return a.n * a.padded <= BP_HELD * BP_THREADS; }
  RTR_DEVICE int held_at(int j) const { return single() ? (tid + j * BP_THREADS) >> 2 : tid + j * BP_THREADS; }
  RTR_DEVICE bool holds(int j) const { return held_at(j) < a.n * (a.padded >> 2); }
  RTR_DEVICE void hold() {
    if (single()) {
#pragma unroll
      for (int j = 0; j < BP_HELD; ++j) {
        const float v = holds(j) ? __ldcg(best + tid + j * BP_THREADS) : -INFINITY;
        held[j] = make_float4(tid & 3 ? -INFINITY : v, (tid & 3) == 1 ? v : -INFINITY, (tid & 3) == 2 ? v : -INFINITY,
                              (tid & 3) == 3 ? v : -INFINITY);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < BP_HELD; ++j)
      if (holds(j)) held[j] = __ldcg(reinterpret_cast<const float4*>(best) + held_at(j));
  }
  // f(row, first group, best logits) for the thread's quartets, of rows that have something to offer: all, or those that are not held
  template <typename F> RTR_DEVICE void each_group(F&& f, int from = 0) const {
    const int quartets = a.padded >> 2, all = a.n * quartets;
    for (int q = tid + from; q < all; q += BP_THREADS) {
      const int r = a.n == 1 ? 0 : row_of((uint32_t)q);
      if (alive(r)) f(r, 4 * (q - r * quartets), __ldcg(reinterpret_cast<const float4*>(best) + q));
    }
  }
  template <typename F> RTR_DEVICE void each_later_group(F&& f) const { each_group(f, BP_HELD * BP_THREADS); }

  // f(row, first place, logits, mask) for the warp's groups of the list
  template <typename F> RTR_DEVICE void each_read(int ng, F&& f) const {
    for (int j = warp; j < ng; j += BP_THREADS / 32) {
      const int id = s.groups[j], r = a.n == 1 ? 0 : row_of((uint32_t)id >> 2), shift = L::shift(row(r));
      const int first = (id - r * a.padded) * L::GROUP - shift, by = MASK ? Allowed<T>::by(mask(r), shift) : 0;
      L raw;
      Allowed<T> ok;
      raw.load(row(r), first, lane, a.vocab);
      if constexpr (MASK) ok.load(mask(r), first, lane, a.vocab, by);
      f(r, first, raw, ok, by);
    }
  }
  // f(row, place in the vocabulary, logit) for the finite, allowed logits of the groups of the list: a group a warp, or a piece a lane at
  // a time (registers that are taken off the usual path are saved on it)
  template <typename F> RTR_DEVICE void each_logit(int ng, F&& f) const {
    each_read(ng, [&](int r, int first, const L& raw, const Allowed<T>& ok, int by) {
#pragma unroll
      for (int i = 0; i < L::EACH; ++i) {
        const float v = raw.one(i);
        if (v > -INFINITY && (!MASK || ok(i, by))) f(r, L::at(first, i, lane), v);
      }
    });
  }
  template <typename F> RTR_DEVICE void each_logit_of_pieces(int ng, F&& f) const {
    for (int i = warp; i < ng * L::PIECES; i += BP_THREADS / 32) {
      const int id = s.groups[i / L::PIECES], r = a.n == 1 ? 0 : row_of((uint32_t)id >> 2);
      const int e = L::at((id - r * a.padded) * L::GROUP - L::shift(row(r)), i % L::PIECES * L::PER, lane);
      each_of_piece(r, e, [&](int j, float x) { f(r, e + j, x); });
    }
  }
  RTR_DEVICE const uint8_t* mask(int r) const { return allowed0 + r * a.allowed_stride; }
  RTR_DEVICE void add(int r, int v, float x) {
    if (near(r, x) > -INFINITY) put(r, v, x);
  }
  RTR_DEVICE void put(int r, int v, float x) {
    const int to = atomicAdd(&s.n_list, 1);
    if (to >= BP_LIST) return;
    s.x[to] = x;
    s.list[to].row = r;
    s.list[to].at = (uint32_t)r * a.vocab + v;
  }

  // Each row's sum from its slices, and what its candidates are offset by: 8 to 32 lanes a row.
  RTR_DEVICE void offsets() {
    static_assert(BP_MAX_N * 8 == BP_THREADS, "a row for every eight threads");
    const int bits = a.n > 64 || a.slices <= 8 ? 3 : a.n > 32 || a.slices <= 16 ? 4 : 5, lanes = 1 << bits, r = tid >> bits, part = tid & (lanes - 1);
    const bool there = r < a.n;
    const float score = there && part == 0 ? a.scores[item * a.n + r] : -INFINITY;
    const float2* p = a.part + ((int64_t)item * a.n + (there ? r : 0)) * a.slices;
    const float2 u = there && part < a.slices ? __ldcg(p + part) : make_float2(-INFINITY, 0.f);
    float all = u.x;
    for (int i = part + lanes; there && i < a.slices; i += lanes) all = fmaxf(all, __ldcg(&p[i].x));
#pragma unroll 1
    for (int d = 1; d < lanes; d <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
    double t = beam_relative(u, all);
#pragma unroll 1
    for (int i = part + lanes; there && i < a.slices; i += lanes) t += beam_relative(__ldcg(p + i), all);
#pragma unroll 1
    for (int d = 1; d < lanes; d <<= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (tid == 0) s.most = s.wild = 0;
    __syncthreads();
    if (there && part == 0) {
      const bool wrong = !(score < INFINITY) || (score > -INFINITY && !(t >= 0.0 && all < INFINITY));
      if (wrong) atomicOr(a.status, RTR_DEV_NAN_SCORE);
      const bool alive = !wrong && score > -INFINITY && all > -INFINITY;
      // log t = exponent log 2 + log of the rest, which is 0.75 to 1.5: a float has that to 2^-25 or so.  (t is relative to a power
      // of two; the sum to the maximum.)
      const float rounded = (float)t;
      const int e = alive ? (int)(__float_as_uint(rounded) - 0x3f400000u) >> 23 : 0;
      const double unit = alive ? beam_offset(all) : 0.0;
      const float rest = alive ? __uint_as_float(__float_as_uint(rounded) - ((uint32_t)e << 23)) : 1.f;
      s.sum[r] = alive ? (e + unit) * 0.69314718055994530942 + (double)(logf(rest) + (float)(t - (double)rounded) / rounded) : 0.0;
      s.off[r] = alive ? (double)score - s.sum[r] : -INFINITY;
      s.near[r] = make_float2(all, (float)s.off[r]);
      s.again[r] = s.done[r] = 0;
      if (alive) atomicMax(&s.most, __float_as_int(fabsf((float)s.off[r])));
      if (alive && fmaxf(all, (float)s.off[r]) > 1e30f) s.wild = 1;
    }
    __syncthreads();
  }

  // A block's share of the sums of the rows marked `again`, in 64 bits: one row after the other, all threads.  The order of a
  // sum goes by places in the vocabulary, not by the row's place in memory, so that equal rows have equal sums.  Of rows that are the
  // same in all places (beams that have not parted yet) one is summed: comparing takes 12 us of
  // 152,704 logits, summing 31.
  RTR_DEVICE void share_again(int rank, int ranks, double (&share)[BP_MAX_N]) {
    for (int r = 0; r < a.n; ++r) {
      if (!s.again[r] || s.done[r]) continue;  // the same for all threads
      const T* p = row(r);
      const float top = s.near[r].x;
      int like = 0;  // the first row of this sum and maximum
      while (like < r && !(s.again[like] && !s.done[like] && s.sum[like] == s.sum[r] && s.near[like].x == top)) ++like;
      if (like < r) {
        const T* q = row(like);
        bool same = true;
        for (int i0 = tid + rank * 8 * BP_THREADS; i0 < a.vocab && same; i0 += ranks * 8 * BP_THREADS) {
          float v[8], w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = i0 + i * BP_THREADS < a.vocab ? to_f32(p[i0 + i * BP_THREADS]) : 0.f;
            w[i] = i0 + i * BP_THREADS < a.vocab ? to_f32(q[i0 + i * BP_THREADS]) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) same &= v[i] == w[i];
        }
        if (__syncthreads_and(same)) {
          if (tid == 0) share[r] = share[like];
          continue;
        }
      }
      const double m = top;
      double part[4] = {0.0, 0.0, 0.0, 0.0};
      for (int i0 = tid + rank * 8 * BP_THREADS; i0 < a.vocab; i0 += ranks * 8 * BP_THREADS) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i0 + i * BP_THREADS < a.vocab ? to_f32(p[i0 + i * BP_THREADS]) : -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i)  // below e^-100 nothing counts: 2^20 of them are 2^-124 of the sum
          part[i & 3] += exp_of(v[i] - top > -100.f ? (double)v[i] - m : -100.0);
      }
      double t = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      if (lane == 0) s.red[warp] = t;
      __syncthreads();
      if (tid == 0) {
        t = 0.0;
        for (int w = 0; w < BP_THREADS / 32; ++w) t += s.red[w];
        share[r] = t;
      }
      __syncthreads();
    }
  }
  RTR_DEVICE void sum_again(int ranks) {
    share_again(0, ranks, s.share[0]);
    if (ranks > 1) cooperative_groups::this_cluster().sync();  // the others' shares are there
    if (tid < a.n && s.again[tid] && !s.done[tid]) {
      double t = 0.0;
      for (int r = 0; r < ranks; ++r) t += s.share[r][tid];
      s.sum[tid] = log(t);
      s.off[tid] = (double)a.scores[item * a.n + tid] - s.sum[tid];
      s.near[tid].y = (float)s.off[tid];
      s.done[tid] = 1;
    }
    __syncthreads();
  }

  // How far below t, which k candidates reach by `near`, others may lie that have to be looked at: what two sums may be off by, and
  // what `near` may (three roundings of 2^-24, with room).
  RTR_DEVICE float slack_of(float t, float most) const { return a.close + 4.77e-7f * (most + fabsf(t)); }
  RTR_DEVICE float slack(float t) const { return slack_of(t, __int_as_float(s.most)); }
  // The same by the rows alone that can have a candidate there (none is worth more than its row's offset): one of a beam
  // at -1e9 leaves no logit of the others out.  Whole warps.
  RTR_DEVICE float least_slack(float t) const {
    float most = 0.f;
    for (int r = lane; r < a.n; r += 32) {
      const float off = s.near[r].y;
      if (off > -INFINITY && off + 4.77e-7f * (fabsf(off) + fabsf(t)) >= t) most = fmaxf(most, fabsf(off));
    }
    return slack_of(t, redux_max(most));
  }

  // What the rows' logits have to reach for `near` to reach t, with room for its roundings.
  RTR_DEVICE void needs(float t) {
    for (int r = tid; r < a.n; r += BP_THREADS) {
      const float2 v = s.near[r];
      s.need[r] = v.y > -INFINITY ? (t - v.y) + v.x - 4.77e-7f * (fabsf(t) + fabsf(v.y) + fabsf(v.x)) : INFINITY;
    }
    __syncthreads();
  }

  // Too few threads have groups for a bound: their lanes' best may give one.
  RTR_DEVICE void needs_by_lanes(int ng) {
    float mine = -INFINITY;
    each_read(ng, [&](int r, int, const L& raw, const Allowed<T>& ok, int by) {
      float x = raw.largest();
      if constexpr (MASK) x = ok.largest(raw, by);
      mine = fmaxf(mine, near(r, x));
    });
    const float t = reached_by(mine, a.k, s);
    needs(t - slack(t));
  }

  // The groups and then the candidates that reach the k-th best of what stands for them: false where there are too many.
  RTR_DEVICE bool gather() {
    if (s.wild) return false;
    if (tid == 0) s.n_quartets = s.n_groups = s.n_whole = s.n_lanes = s.n_list = 0;
    float mine = -INFINITY, of[BP_HELD];  // of: the held quartets' best
#pragma unroll
    for (int j = 0; j < BP_HELD; ++j) {
      const int r = !holds(j) || a.n == 1 ? 0 : row_of((uint32_t)held_at(j));
      const float x = fmaxf(fmaxf(held[j].x, held[j].y), fmaxf(held[j].z, held[j].w));
      of[j] = holds(j) && alive(r) ? near(r, x) : -INFINITY;
      mine = fmaxf(mine, of[j]);
    }
    each_later_group([&](int r, int, const float4& v) {
      mine = fmaxf(mine, near(r, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))));
    });
    const float t = reached_by(mine, a.k, s), floor_ = t - slack(t);
    needs(floor_);
    const auto put = [&](int q, const float4& v) {
      const int to = atomicAdd(&s.n_quartets, 1);
      if (to >= BP_GROUPS) return;
      s.quartet[to] = v;
      s.quartet_at[to] = q;
    };
    if (mine > -INFINITY && mine >= floor_) {
#pragma unroll
      for (int j = 0; j < BP_HELD; ++j)
        if (of[j] > -INFINITY && of[j] >= floor_) put(held_at(j), held[j]);
      each_later_group([&](int r, int g0, const float4& v) {
        if (near(r, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))) >= floor_) put((r * a.padded + g0) >> 2, v);
      });
    }
    __syncthreads();
    const int nq = s.n_quartets;
    if (nq > BP_GROUPS) return false;
    for (int i = tid; i < 4 * nq; i += BP_THREADS) {
      const int q = s.quartet_at[i >> 2], r = a.n == 1 ? 0 : row_of((uint32_t)q);
      const float v = (&s.quartet[i >> 2].x)[i & 3];
      if (v >= s.need[r] && v > -INFINITY) {
        const int to = atomicAdd(&s.n_groups, 1);
        if (to < BP_GROUPS) s.groups[to] = 4 * q + (i & 3);
      }
    }
    __syncthreads();
    const int ng = s.n_groups;
    if (ng > BP_GROUPS) return false;
    if (!(t > -INFINITY) && ng > 1) pick_needs<T, MASK>(a, s, ng);
    // Hardly ever more than one lane of a group has any, and the first kernel has said which.  Of other groups all lanes are
    // looked at, or, where there are many, those whose largest logit says so.
    int whole = -1, r = 0, first = 0;
    if (tid < ng) {
      const int id = s.groups[tid];
      r = a.n == 1 ? 0 : row_of((uint32_t)id >> 2);
      first = (id - r * a.padded) * L::GROUP - L::shift(row(r));
      const uint32_t w = __ldcg(a.second + ((int64_t)item * a.n * a.padded + id));
      if (beam_second_value(w) < s.need[r]) add_lane(r, first, (int)(w & 31));
      else whole = id;
    }
    const int wholes = __syncthreads_count(whole >= 0);
    if (ng + 31 * wholes <= BP_LANES) {
      if (whole >= 0) {
        const int to = atomicAdd(&s.n_lanes, 32);
        for (int l = 0; l < 32; ++l) s.lane[to + l] = make_int2(32 * r + l, first);
      }
    } else {
      if (whole >= 0) s.groups[atomicAdd(&s.n_whole, 1)] = whole;
      __syncthreads();
      pick_whole<T, MASK>(a, s);
    }
    __syncthreads();
    const int nl = s.n_lanes;
    if (nl > BP_LANES) return false;
    for (int i = tid; i < nl * L::PIECES; i += BP_THREADS) {
      const int2 l = s.lane[i / L::PIECES];
      r = l.x >> 5;
      const int e = L::at(l.y, i % L::PIECES * L::PER, l.x & 31);
      const float x = s.need[r];
      each_of_piece(r, e, [&](int j, float v) {
        if (v >= x) add(r, e + j, v);
      });
    }
    __syncthreads();
    return s.n_list <= BP_LIST;
  }
  // f(j, logit) for the finite, allowed logits of row r's piece at place e of the vocabulary
  template <typename F> RTR_DEVICE void each_of_piece(int r, int e, F&& f) const {
    const uint4 u = e >= 0 && e + L::PER <= a.vocab ? __ldg(reinterpret_cast<const uint4*>(row(r) + e)) : beam_ragged(row(r), e, a.vocab);
    bool ok[L::PER];
    if constexpr (MASK) {
#pragma unroll
      for (int j = 0; j < L::PER; ++j) ok[j] = e + j >= 0 && e + j < a.vocab && mask(r)[e + j];
    }
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < L::PER; ++j) {
      const float v = __uint_as_float(sizeof(T) == 4 ? w[j % 4] : j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
      if (v > -INFINITY && (!MASK || ok[j])) f(j, v);
    }
  }
  RTR_DEVICE void add_lane(int r, int first, int lane_) {
    const int to = atomicAdd(&s.n_lanes, 1);
    if (to < BP_LANES) s.lane[to] = make_int2(32 * r + lane_, first);
  }
  RTR_DEVICE void take_whole() {
    each_read(s.n_whole, [&](int r, int first, const L& raw, const Allowed<T>&, int) {
      if (raw.largest() >= s.need[r]) add_lane(r, first, lane);
    });
  }

  // Where these are too many the bound was too low: threads stand for several groups, so where most of the k best are
  // candidates of few rows (the other beams are far behind), a row of another has the k-th best thread.  Here every group counts, and then
  // every logit of the groups that reach the bound; false where there are too many still (ties).  (50 beams of 152,704, one 6 or more
  // ahead of the others: 49 - 52 us a call; with each row's sum in 64 bits and the exact search below 2,680.)
  RTR_DEVICE bool gather_closely() {
    if (s.wild) return false;
    const auto groups = [&](auto&& f) {
      each_group([&](int r, int g0, const float4& v) {
        f(near(r, v.x), r, g0);
        f(near(r, v.y), r, g0 + 1);
        f(near(r, v.z), r, g0 + 2);
        f(near(r, v.w), r, g0 + 3);
      });
    };
    const auto by_groups = [&](auto&& f) { groups([&](float v, int, int) { f(v); }); };
    const auto too_many = [&](float least) {  // or the list of those that reach it
      if (tid == 0) s.n_groups = 0;
      __syncthreads();
      groups([&](float v, int r, int g) {
        if (!(v > -INFINITY) || v < least || so_far(s.n_groups) > BP_GROUPS) return;
        const int to = atomicAdd(&s.n_groups, 1);
        if (to < BP_GROUPS) s.groups[to] = r * a.padded + g;
      });
      __syncthreads();
      return s.n_groups > BP_GROUPS;
    };
    const auto logits = [&](float least, auto&& f) {
      each_logit_of_pieces(s.n_groups, [&](int r, int at, float x) {
        if (near(r, x) >= least) f(r, at, x);
      });
    };
    const auto by_logits = [&](float least) {
      return [&, least](auto&& f) { logits(least, [&](int r, int, float x) { f(near(r, x)); }); };
    };
    float t = reached_among<false>(by_groups, a.k, s);
    const uint32_t top = __reduce_max_sync(0xffffffffu, s.word[lane]);  // the largest of all, of groups or logits
    if (too_many(t - least_slack(t))) {
      if (float_key(t) >= top) return false;
      // the groups above the k-th one's bin, fewer than k, may have k logits; or a closer look at the groups shows that fewer will do
      const uint32_t above = s.above;
      too_many(nextafterf(key_float(above), INFINITY));
      if (tid == 0) s.above = top;
      t = fmaxf(t, reached_among<true>(by_logits(-INFINITY), a.k, s));
      bool many = too_many(t - least_slack(t));
      if (many && tid == 0) s.above = above;
      for (int i = 0; i < 2 && many; ++i) {
        t = fmaxf(t, reached_among<true>(by_groups, a.k, s));
        many = too_many(t - least_slack(t));
      }
      if (many) return false;
    }
    const float least = t - least_slack(t);
    if (tid == 0) s.above = top;
    for (int i = 0; i < 2; ++i) {
      t = fmaxf(t, reached_among<true>(by_logits(least), a.k, s));
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      logits(t - least_slack(t), [&](int r, int at, float x) {
        if (so_far(s.n_list) <= BP_LIST) add(r, at, x);
      });
      __syncthreads();
      if (s.n_list <= BP_LIST) return true;
      if (float_key(t) >= top) return false;
      __syncthreads();
    }
    return false;
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
  // value's 64 bits and, among equal ones, of the place.  Rows are summed in 64 bits first.
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
  RTR_DEVICE void gather_exactly() {
    for (int r = tid; r < a.n; r += BP_THREADS) s.again[r] = a.n > 1 && s.off[r] > -INFINITY;
    __syncthreads();
    sum_again(1);
    uint64_t least;
    uint32_t last;
    const auto groups = [&](auto&& f) {
      each_group([&](int r, int g0, const float4& v) {
        const float w[4] = {v.x, v.y, v.z, v.w};
        for (int i = 0; i < 4; ++i)
          if (w[i] > -INFINITY && g0 + i < a.groups && counts(worth(r, w[i]))) f(double_key(worth(r, w[i])), (uint32_t)(r * a.padded + g0 + i));
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
    const auto logits = [&](auto&& f) {  // the same ones in every pass: so no more than k are added
      each_logit(ng, [&](int r, int v, float x) {
        const double value = worth(r, x);
        if (counts(value)) f(double_key(value), (uint32_t)r * a.vocab + v, r, v, x);
      });
    };
    bisect([&](auto&& f) { logits([&](uint64_t key, uint32_t at, int, int, float) { f(key, at); }); }, a.k, least, last);
    logits([&](uint64_t key, uint32_t at, int r, int v, float x) {
      if (key > least || (key == least && at < last)) put(r, v, x);
    });
    __syncthreads();
  }

  // Candidates by value, then place: each one's rank is the number of those before it, counted by eight threads.  (110 candidates
  // 2,500 cycles; a bitonic sort by shuffles 7,500.)
  RTR_DEVICE void put_in_order() {
    const int n = s.n_list;
    for (int i = tid; i < n; i += BP_THREADS) s.list[i].key = double_key(worth(s.list[i].row, s.x[i]));
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += BP_THREADS / 8) {
      const int i = i0 + (tid >> 3);
      int before = 0;
      if (i < n) {
        const PickEntry me = s.list[i];
        for (int j = tid & 7; j < n; j += 8) {
          const PickEntry it = s.list[j];
          before += (it.key > me.key) | ((it.key == me.key) & (it.at < me.at));
        }
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
      if (i < n && (tid & 7) == 0) s.order[before] = (uint16_t)i;
    }
    __syncthreads();
  }

  // Marks the rows of candidates among (or just behind) the first k that are too close to those of another row, rows
  // of one 32-bit sum among them: what tells them apart may be too small for it.
  RTR_DEVICE bool doubtful() {
    const int n = s.n_list;
    bool doubt = false;
    for (int i = tid; i + 1 < n; i += BP_THREADS) {
      // behind the k-th everything is compared with that one
      const PickEntry p = s.list[s.order[min(i, a.k - 1)]], q = s.list[s.order[i + 1]];
      const int rp = p.row, rq = q.row;
      if (rp == rq || (s.done[rp] && s.done[rq])) continue;
      if (key_double(p.key) - key_double(q.key) >= a.close) continue;
      s.again[rp] = s.again[rq] = 1;
      doubt = true;
    }
    return __syncthreads_or(doubt);
  }
  RTR_DEVICE void settle() {
    if (tid == 0) s.doubt = 1;
    if (a.ranks > 1) cooperative_groups::this_cluster().sync();  // the others may look
    sum_again(a.ranks);
    put_in_order();
  }
};

template <typename T, bool MASK> RTR_DEVICE Picker<T, MASK> picker(const BeamPick& a, PickShared& s) {
  const int tid = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * a.n;
  return Picker<T, MASK>{a, s, (int)blockIdx.x, tid, tid >> 5, tid & 31, static_cast<const T*>(a.logits) + row0 * a.stride,
                         MASK ? a.allowed + row0 * a.allowed_stride : nullptr, a.best + row0 * a.padded, {}};
}
template <typename T, bool MASK> __device__ __noinline__ void pick_closely(const BeamPick& a, PickShared& s) {
  if (!picker<T, MASK>(a, s).gather_closely()) pick_exactly<T, MASK>(a, s);
}
template <typename T, bool MASK> __device__ __noinline__ void pick_exactly(const BeamPick& a, PickShared& s) {
  picker<T, MASK>(a, s).gather_exactly();
}
template <typename T, bool MASK> __device__ __noinline__ void pick_needs(const BeamPick& a, PickShared& s, int ng) {
  picker<T, MASK>(a, s).needs_by_lanes(ng);
}
template <typename T, bool MASK> __device__ __noinline__ void pick_whole(const BeamPick& a, PickShared& s) {
  picker<T, MASK>(a, s).take_whole();
}
template <typename T, bool MASK> __device__ __noinline__ void pick_again(const BeamPick& a, PickShared& s) {
  picker<T, MASK>(a, s).settle();
}
// The other blocks of an item's cluster: they wait for the first one's doubts, and take their shares of the sums.
template <typename T, bool MASK> RTR_DEVICE void pick_help(const BeamPick& a, PickShared& s) {
  const auto cluster = cooperative_groups::this_cluster();
  const int tid = threadIdx.x, rank = (int)cluster.block_rank();
  cluster.sync();
  PickShared* lead = cluster.map_shared_rank(&s, 0);
  if (lead->doubt) {
    if (tid < a.n) {
      s.again[tid] = lead->again[tid];
      s.done[tid] = lead->done[tid];
      s.sum[tid] = lead->sum[tid];
      s.near[tid].x = lead->near[tid].x;
    }
    __syncthreads();
    picker<T, MASK>(a, s).share_again(rank, a.ranks, lead->share[rank]);
    cluster.sync();
  }
  cluster.sync();  // the first block does not leave before its flag is read
}
// Fewer finite candidates than k: the first places that have none.
__device__ __noinline__ void pick_fill(const BeamPick& a, PickShared& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = s.n_list;
  const int64_t all = (int64_t)a.n * a.vocab;
  bool free_ = tid < 2 * a.k && tid < all;
  for (int j = 0; j < n && free_; ++j) free_ = s.list[j].at != (uint32_t)tid;
  const unsigned mask = __ballot_sync(0xffffffffu, free_);
  if (lane == 0) s.red[warp] = __popc(mask);
  __syncthreads();
  int before = __popc(mask & ((1u << lane) - 1));
  for (int w = 0; w < warp; ++w) before += (int)s.red[w];
  if (free_ && n + before < a.k) {
    s.list[n + before] = PickEntry{double_key(-INFINITY), (uint32_t)tid, (uint32_t)(tid / a.vocab)};
    s.order[n + before] = (uint16_t)(n + before);
  }
  __syncthreads();
}

// HELP: a cluster of a.ranks blocks an item, else one block.
template <typename T, bool MASK, bool HELP>
__global__ void __launch_bounds__(BP_THREADS) beam_pick_kernel(const __grid_constant__ BeamPick a) {
  __shared__ PickShared s;
  pdl_launch_dependents();
  pdl_wait();
  const int item = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if constexpr (HELP)
    if (blockIdx.z) {
      pick_help<T, MASK>(a, s);
      return;
    }
  Picker<T, MASK> p = picker<T, MASK>(a, s);
  p.hold();
  p.offsets();
  if (!p.gather()) pick_closely<T, MASK>(a, s);
  p.put_in_order();
  if (p.doubtful()) {
    pick_again<T, MASK>(a, s);
  } else if constexpr (HELP) {
    if (tid == 0) s.doubt = 0;
    cooperative_groups::this_cluster().sync();
  }
  if (s.n_list < a.k) pick_fill(a, s);
  if (tid < a.k) {
    const PickEntry c = s.list[s.order[tid]];
    const int64_t to = (int64_t)item * a.k + tid;
    a.all_tokens[to] = (int32_t)(c.at - c.row * a.vocab);
    a.all_parents[to] = (int32_t)c.row;
    a.all_scores[to] = (float)key_double(c.key);
  }
  if (warp == 0) {
    int taken = 0;
    for (int j0 = 0; j0 < a.k && taken < a.beams; j0 += 32) {
      const int j = j0 + lane;
      const PickEntry c = s.list[s.order[min(j, a.k - 1)]];
      const int token = (int32_t)(c.at - c.row * a.vocab);
      const bool on = j < a.k && token != a.eos;
      const unsigned mask = __ballot_sync(0xffffffffu, on);
      const int place = taken + __popc(mask & ((1u << lane) - 1));
      if (on && place < a.beams) {
        const int64_t to = (int64_t)item * a.beams + place;
        a.next_tokens[to] = token;
        a.next_parents[to] = (int32_t)c.row;
        a.next_scores[to] = (float)key_double(c.key);
      }
      taken += __popc(mask);
    }
  }
  if constexpr (HELP) cooperative_groups::this_cluster().sync();
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

// Values of different rows may be told wrong by their sums of 32 bits where they are closer than this: twice what the log of one
// such sum may be off by, whatever the logits.  In units of 2^-24:
//  - exponents y round by |y| at most, and |y| <= 8.5 + max(0, D - 16) with D the distance from the row's maximum in units of log2.  The
//    mean of that over a row, whose weights are 2^-D / sum, is at most 9.95 + max(0, log2(vocab) - 17.44): where w of the weight lies beyond
//    16, the mean of D there is at most log2(vocab) - log2(w), since nothing over vocab places has an entropy above log(vocab).  Times log 2;
//  - a group's additions: 3 + 2 in bf16, 1 + 2 in fp32, and twice one where a group is more than all before it;
//  - a slice's sum rounded to a float: 1; the logarithm of the rest: 0.75.
// And what errs to one side, once: ex2.approx is off by -1.45e-7 to 1.46e-7 (all floats from -40 to 40 measured), log2(e) as a float by
// 1.34e-8 of the exponent.  For 152,832 logits 2.3e-6 in bf16, 2.1e-6 in fp32.
static float beam_close(int vocab, bool fp32) {
  const float spread = std::log((float)vocab);
  const float one = 6.9f + std::max(0.f, spread - 12.08f) + (fp32 ? 3.f : 5.f) + 2.f + 1.75f;
  return 2.f * 5.97e-8f * one + 2.92e-7f + 1.34e-8f * spread;
}

// Groups of a row (one more where it starts in the middle of one), slices, and the workspace they need.
static void beam_plan(const rtr_beam_step* b, int sms, BeamPick& p, int64_t& groups_bytes, int64_t& bytes) {
  const int per = b->dtype == RTR_DTYPE_F32 ? 4 : 8;
  const int group = BP_BYTES * per / 16;
  p.groups = (int)(((int64_t)b->vocab + per - 1 + group - 1) / group);
  p.padded = (p.groups + 3) & ~3;
  p.quarter_inv = (uint32_t)((0x100000000ull + p.padded / 4 - 1) / (p.padded / 4));
  // Slices of a row: enough for as many blocks as the SMs hold at once where the rows are few (a warp takes a group at least), and eight
  // times as many blocks as that where they are many.  200 rows of 152,832 in bf16: 2, 3, 4 slices 24.9, 21.5, 22.4 us; 50 of 152,704 in
  // fp32: 8, 11, 16 slices 14.9, 14.3, 15.0; 1,600 rows: 1 to 4 slices the same.
  const int64_t rows = (int64_t)b->items * b->n, room = beam_blocks(b->allowed != nullptr) * (int64_t)sms;
  const int64_t want = ((rows <= room ? room : 8 * room) + rows - 1) / std::max<int64_t>(rows, 1);
  const int64_t slices = std::max<int64_t>(1, std::min<int64_t>(want, (p.groups + BP_WARPS - 1) / BP_WARPS));
  p.slices = (int)slices;
  groups_bytes = rows * p.padded * (int64_t)sizeof(float);  // a multiple of 16
  bytes = 2 * groups_bytes + rows * p.slices * (int64_t)sizeof(float2);
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
  p.close = beam_close(step->vocab, step->dtype == RTR_DTYPE_F32);
  p.best = static_cast<float*>(workspace);
  p.second = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + best);
  p.part = reinterpret_cast<float2*>(static_cast<char*>(workspace) + 2 * best);
  p.all_tokens = step->all_tokens;
  p.all_parents = step->all_parents;
  p.all_scores = step->all_scores;
  p.next_tokens = step->next_tokens;
  p.next_parents = step->next_parents;
  p.next_scores = step->next_scores;
  p.status = step->status;
  // Where there are eight items or more, of two rows at least (one row is never in doubt), an item is in doubt now and then (one in 80
  // or so), and summing its rows takes one block long where they are long (65,536 logits 14 us each): its block has others of a
  // cluster beside it, on SMs that have no item.  (One block : four, us, 24 calls.  16 items of 10 rows: of 32,003 without doubts 13.2 :
  // 14.4, of 65,536, one with, 14.6 : 15.7, in the mean 15.7 : 16.2, and that one 41 : 27.  32 of 50 rows in the mean: of 32,003 49.8 : 49.7, of
  // 65,536 60.3 : 58.5, of 131,072 96.2 : 87.4.)
  p.ranks = 1;
  if (step->items >= 8 && step->n > 1 && step->vocab >= 1 << 16)
    while (p.ranks < BP_RANKS && 2 * p.ranks * (int64_t)step->items <= on.sms) p.ranks *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto run = [&](auto scan, auto pick) {
    const cudaError_t e = kv_launch(scan, dim3((unsigned)blocks), BP_WARPS * 32, 0, 1, st, p);
    return e == cudaSuccess ? kv_launch(pick, dim3((unsigned)p.items, 1, (unsigned)p.ranks), BP_THREADS, 0, p.ranks, st, p) : e;
  };
  const auto run_type = [&](auto type, auto mask) {
    using T = decltype(type);
    constexpr bool MASK = decltype(mask)::value;
    return p.ranks > 1 ? run(beam_scan_kernel<T, MASK>, beam_pick_kernel<T, MASK, true>)
                       : run(beam_scan_kernel<T, MASK>, beam_pick_kernel<T, MASK, false>);
  };
  cudaError_t e;
  if (step->dtype == RTR_DTYPE_F32) e = p.allowed ? run_type(float{}, std::true_type{}) : run_type(float{}, std::false_type{});
  else e = p.allowed ? run_type(__nv_bfloat16{}, std::true_type{}) : run_type(__nv_bfloat16{}, std::false_type{});
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
