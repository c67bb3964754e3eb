// Decode attention over a kept prefix: what the attention over the 8-bit cache's pages
// gave for the prefix (out and the log of its softmax sum) joined with the beams' own
// tokens, at most four, found through the ancestry table as in attention.cu.
//
//   out = (e^lse out_p + sum_j e^{s_j} v_j) / (e^lse + sum_j e^{s_j}),  s_j = scale q . k_j
//
// relative to the largest exponent.  A warp takes one (beam, head); 50 beams x 28 heads
// move under 2 MB, so the launch bounds it.
#include "common.cuh"
#include "engine.h"

namespace rtr {

constexpr int KS_WARPS = 8;

template <typename T, int D>
__global__ void __launch_bounds__(KS_WARPS * 32) kv_suffix_kernel(
    const T* __restrict__ q, const T* __restrict__ prefix, const float* __restrict__ lse, const T* __restrict__ ksuf,
    const T* __restrict__ vsuf, const int32_t* __restrict__ anc, int t, T* __restrict__ out,
    float* __restrict__ out_big, float* __restrict__ out_small, int beams, int heads, int kv_heads, float scale,
    uint32_t* __restrict__ status, int xfmt) {
  constexpr int PER = D / 32;
  const int i = blockIdx.x * KS_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= beams * heads) return;
  const int b = i / heads, h = i % heads, g = h / (heads / kv_heads);
  const long at = (long)i * D + lane * PER;
  float x[PER], o[PER], s[4], v[4][PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) x[j] = to_f32(q[at + j]);
  const float lp = lse[i];
  float m = lp;
#pragma unroll
  for (int sl = 0; sl < 4; ++sl) {
    s[sl] = -INFINITY;
    if (sl >= t) continue;
    int row = sl == t - 1 ? b : anc[b * 4 + sl];
    if (row < 0 || row >= beams) {
      if (lane == 0) atomicOr(status, RTR_DEV_BAD_PARENT);
      row = b;
    }
    const long from = (((long)sl * beams + row) * kv_heads + g) * D + lane * PER;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      dot = fmaf(x[j], to_f32(ksuf[from + j]), dot);
      v[sl][j] = to_f32(vsuf[from + j]);
    }
    s[sl] = warp_sum(dot) * scale;
    m = fmaxf(m, s[sl]);
  }
  const float wp = lp == -INFINITY ? 0.f : expf(lp - m);
  float sum = wp;
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = wp * to_f32(prefix[at + j]);
#pragma unroll
  for (int sl = 0; sl < 4; ++sl) {
    if (sl >= t) continue;
    const float w = expf(s[sl] - m);
    sum += w;
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = fmaf(w, v[sl][j], o[j]);
  }
  const float inv = 1.0f / sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if constexpr (sizeof(T) == 4) store_split(out, out_big, out_small, at + j, o[j] * inv, xfmt);
    else out[at + j] = from_f32<T>(o[j] * inv);
  }
}

template <typename T>
static cudaError_t launch(const void* q, const void* prefix, const float* lse, const void* ks, const void* vs,
                          const int32_t* anc, int t, void* out, float* big, float* small, int beams, int heads,
                          int kv_heads, int head_dim, float scale, uint32_t* status, int xfmt, cudaStream_t st) {
  const unsigned blocks = (unsigned)((beams * heads + KS_WARPS - 1) / KS_WARPS);
  const auto run = [&](auto kernel) {
    kernel<<<blocks, KS_WARPS * 32, 0, st>>>(static_cast<const T*>(q), static_cast<const T*>(prefix), lse,
                                             static_cast<const T*>(ks), static_cast<const T*>(vs), anc, t,
                                             static_cast<T*>(out), big, small, beams, heads, kv_heads, scale, status,
                                             xfmt);
    return cudaGetLastError();
  };
  return head_dim == 128 ? run(kv_suffix_kernel<T, 128>) : run(kv_suffix_kernel<T, 64>);
}

cudaError_t kv_suffix_join(const void* q, const void* prefix, const float* lse, const void* k_suffix,
                           const void* v_suffix, const int32_t* anc, int t, void* out, float* out_big,
                           float* out_small, int beams, int heads, int kv_heads, int head_dim, float scale,
                           uint32_t* status, bool bf16, int xfmt, cudaStream_t stream) {
  if (bf16)
    return launch<__nv_bfloat16>(q, prefix, lse, k_suffix, v_suffix, anc, t, out, out_big, out_small, beams, heads,
                                 kv_heads, head_dim, scale, status, xfmt, stream);
  return launch<float>(q, prefix, lse, k_suffix, v_suffix, anc, t, out, out_big, out_small, beams, heads, kv_heads,
                       head_dim, scale, status, xfmt, stream);
}

}  // namespace rtr
