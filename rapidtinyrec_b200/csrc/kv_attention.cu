// Attention over the 8-bit KV cache: softmax(scale q K^T) V of new query rows
// over sequences whose K and V are e4m3 codes in pages, with one scale a page.
//
// Mathematics.  With codes c and scales s the score of key j is
// scale * s_k(page of j) * (q . ck_j); the scale multiplies the finished dot
// product, so the codes enter the matrix instructions as they are (e4m3 is exact
// in fp16).  One pass over the keys keeps, per row, a running maximum M of
// score * log2(e) + log2(s_v), the weights w_j = 2^(score log2(e) + log2 s_v - M),
// the sum of w_j cv_j and the softmax's own sum of w_j / s_v: the V scale costs an
// addition in the exponent, every weight is at most 1 whatever the scales are,
// and both sums end up relative to the same M.
//
// Rows.  The query rows of one KV head are its (token, head of the group) pairs.
// A block takes a tile of them and a stretch of the sequence's keys; the keys are
// split over blocks while there are fewer tiles than the GPU has room for.  Up to
// eight stretches are a thread-block cluster, whose blocks join their sums through
// distributed shared memory; more are joined by a second kernel.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "engine.h"
#include "kv_attention.cuh"
#include "kv_host.h"
#include "tcgen05.cuh"

namespace rtr {

constexpr int KA_WARPS = 4, KA_ROWS = 8, KA_KEYS = 32, KA_STAGES = 2;
constexpr int KA_MAX_CHUNK = 1024;  // 16 16-key segments a warp: their page numbers and scales fit its lanes
template <int D> struct KaCfg {
  static constexpr int STAGE = 2 * KA_KEYS * D;  // K and V of one key group
  static constexpr int WARP_BYTES = KA_STAGES * STAGE;
  static constexpr int LD = D + 4;               // row of the joining buffer, floats
  static constexpr int RING = KA_WARPS * WARP_BYTES;
  static constexpr int JOIN = KA_WARPS * KA_ROWS * LD * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

RTR_DEVICE void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same, from zeros.
RTR_DEVICE void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {z, z, z, z};\n\t}"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
RTR_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// Where 16-byte piece `ch` of key row `row` lies in a stage: pieces are permuted
// within 128 bytes so that the rows g, g + 1 that eight lanes read of K, and the
// rows 0, 2, 4, 6 (or 1, 3, 5, 7) that they read of V, lie in different banks.
template <int D> RTR_DEVICE int ka_at(int row, int ch) {
  if constexpr (D == 128) {
    return row * 128 + ((ch ^ (row & 6) ^ ((row & 1) << 2)) << 4);
  } else {
    const int line = row >> 1;
    return line * 128 + (((((row & 1) << 2) + ch) ^ ((line & 3) << 1)) << 4);
  }
}

// One block: KA_ROWS query rows, up to `chunk` keys.  Its warps take 32-key groups
// in turn, each with its own running maximum, and are joined at the end.
//
// The products are transposed (keys as the 16 rows of an m16n8k16, query rows as
// its 8 columns), so a group of up to 8 query heads fills the instruction.  Which
// dimension sits where in a contraction is free, as long as both operands agree:
// a lane takes 16 consecutive codes of a key for q . k and, of the keys it needs
// for P V, 16 consecutive dimensions, so both operands come from shared memory by
// 16-byte loads and the transposition of V is byte permutes in registers.
//
// fp32 queries (and weights) enter as fp16 pairs, hi + lo: 22 significant bits.  The weights' low
// parts have a product of their own, times KA_LOW, which is added to the sums by IEEE operations.
template <typename T, int D>
__global__ void __launch_bounds__(KA_WARPS * 32, 3) kv_attn_rows_kernel(const KvAttn a) {
  using C = KaCfg<D>;
  constexpr bool PAIR = std::is_same<T, float>::value;
  constexpr int KW = D / 16;   // 4-code words of a key a lane holds: one q . k instruction each
  constexpr int VW = D / 32;   // words of a V row a lane holds
  constexpr int DG = D / 8;    // dimensions of the output a lane holds, for two rows
  extern __shared__ __align__(128) uint8_t ka_smem[];
  __shared__ int slot[2];
  __shared__ float join_m[KA_WARPS][KA_ROWS], join_l[KA_WARPS][KA_ROWS];
  __shared__ __align__(16) float sum_o[KA_ROWS][D];  // this block's sums, read by its cluster
  __shared__ float2 sum_ml[KA_ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y, split = blockIdx.z;
  pdl_launch_dependents();
  pdl_wait();

  int seq;
  int64_t item0;
  if (a.b.starts) {
    seq = kv_find_seq(a.b, blockIdx.x, a.group, 3, 1, a.c.status, slot, item0);
    if (a.refused && tid == 0) *a.refused = seq == -2;  // every block says the same
    if (seq < 0) return;
  } else {
    seq = (int)blockIdx.x / a.per_seq;
    item0 = (int64_t)seq * a.per_seq;
  }
  // What needs no other load's result is loaded first: the length, this lane's page
  // number and its part of the query rows.
  int first, count, len = a.b.lens[seq];
  if (!kv_rows(a.b, seq, a.c.status, first, count)) return;
  const int nrows = count * a.group, r0 = (int)(blockIdx.x - item0) * KA_ROWS;
  if (r0 >= nrows) return;
  const int c0 = split * a.chunk;
  // lane 2 i + h: the h-th 16 keys of this warp's i-th group (a page is a multiple of 16)
  const int key_at = c0 + KA_KEYS * (warp + KA_WARPS * (lane >> 1)) + 16 * (lane & 1);
  const int page = a.b.table[(int64_t)seq * a.b.table_stride + min(key_at >> a.c.page_shift, a.b.table_width - 1)];
  uint4 raw[D * sizeof(T) / 64];  // dimensions 16 c .. 16 c + 15 (and 64 more) of query row g
  {
    const int row = r0 + g, token = row / a.group;
    const T* p = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.q_token +
                 (int64_t)(kvh * a.group + row - token * a.group) * D + 16 * c;
    constexpr int PER = sizeof(T);  // 16-byte loads of 16 values
#pragma unroll
    for (int i = 0; i < D / 64 * PER; ++i)
      raw[i] = row < nrows ? *reinterpret_cast<const uint4*>(p + 64 * (i / PER) + 16 / PER * (i % PER))
                           : make_uint4(0u, 0u, 0u, 0u);
  }
  const bool whole = kv_len_fits(a.c, a.b, len, 0);
  if (!whole) len = 0;  // the sequence's rows become NaN
  // keys that a row of token t sees
  const auto limit = [&](int row) {
    return a.causal && count > 1 ? max(0, len - count + min(row, nrows - 1) / a.group + 1) : len;
  };
  const int kmin = limit(r0), kmax = limit(r0 + KA_ROWS - 1);
  const int c1 = min(kmax, c0 + a.chunk);
  if (c1 <= c0 && split > 0 && !a.cluster) {  // a stretch behind the last key (the first one reports rows that see nothing)
    if (tid < KA_ROWS && r0 + tid < nrows) {
      const int rr = r0 + tid;
      const int64_t rh = (int64_t)(first + rr / a.group) * a.heads + kvh * a.group + rr % a.group;
      a.ml[rh * a.splits + split] = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  const int groups = c1 > c0 ? (c1 - c0 + KA_KEYS - 1) / KA_KEYS : 0;
  const int n = (groups - warp + KA_WARPS - 1) / KA_WARPS;  // this warp's groups: warp, warp + 4, ...

  int64_t at = kvh * a.c.head_stride;
  float ks = 0.f, vs = 0.f;  // where there are no keys: scores are masked
  if (key_at < c1) {
    if (page >= 0 && page < a.c.pages) {
      at += page * a.c.page_stride + (int64_t)(key_at & ((1 << a.c.page_shift) - 1)) * D;
      ks = a.c.k_scale[page * a.c.scale_stride + kvh];
      vs = a.c.v_scale[page * a.c.scale_stride + kvh];
    } else {
      atomicOr(a.c.status, RTR_DEV_BAD_PAGE);
      ks = __int_as_float(0x7fffffff);  // the rows that see the page become NaN
    }
  }
  uint8_t* ring = ka_smem + warp * C::WARP_BYTES;
  const auto issue = [&](int i) {
    if (i < n) {
      const int left = c1 - (c0 + KA_KEYS * (warp + KA_WARPS * i));
      uint8_t* st = ring + (i % KA_STAGES) * C::STAGE;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t from = __shfl_sync(0xffffffffu, at, 2 * i + h) + 16 * lane;
        const uint8_t *k = a.c.k + from, *v = a.c.v + from;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const int x = lane + 32 * j, row = 16 * h + x / (D / 16), ch = x % (D / 16);
          const bool there = row < left;  // keys behind the last are zeros
          cp_async16(st + ka_at<D>(row, ch), k + 512 * j, there);
          cp_async16(st + KA_KEYS * D + ka_at<D>(row, ch), v + 512 * j, there);
        }
      }
    }
    cp_async_commit();
  };
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < KA_STAGES - 1; ++i) issue(i);
  }

  float lvs = 0.f, ivs = 0.f;
  if (key_at < c1) {
    ks = kv_k_scale(ks);
    kv_v_scale(vs, lvs, ivs);
  }

  // the query rows as fp16 times a power of two that puts a row's largest value into [2^13, 2^14)
  uint32_t qh[KW][2], ql[PAIR ? KW : 1][2];
  float f0, f1;  // back to the score, in units of log2, for rows 2 c and 2 c + 1
  {
    float x[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      const uint4& u = raw[i * sizeof(T) / 16];
      const uint32_t w = (&u.x)[i * sizeof(T) % 16 / 4];
      if constexpr (PAIR) x[i] = __uint_as_float(w);
      else x[i] = __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = kv_row_exponent(top);
    const float up = kv_pow2(-e), back = kv_pow2(e) * a.factor;
    f0 = __shfl_sync(0xffffffffu, back, 8 * c);
    f1 = __shfl_sync(0xffffffffu, back, 8 * c + 4);
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float u = x[4 * w + 2 * h] * up, v = x[4 * w + 2 * h + 1] * up;
        qh[w][h] = pack_f16(u, v);
        if constexpr (PAIR) {
          const float2 r = rest_f16(qh[w][h], u, v);
          ql[w][h] = pack_f16(r.x, r.y);
        }
      }
  }
  const int lim0 = limit(r0 + 2 * c), lim1 = limit(r0 + 2 * c + 1);

  float o[DG / 2][4];  // [dims 2 j, 2 j + 1 of this lane's][row 2 c, row 2 c + 1]
#pragma unroll
  for (int j = 0; j < DG / 2; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  for (int i = 0; i < n; ++i) {
    cp_async_wait<KA_STAGES - 2>();
    __syncwarp();
    issue(i + KA_STAGES - 1);  // into the stage that every lane has read in the last round
    const uint8_t* kst = ring + (i % KA_STAGES) * C::STAGE;
    const uint8_t* vst = kst + KA_KEYS * D;
    const int key0 = c0 + KA_KEYS * (warp + KA_WARPS * i);
    float iv[2];

    // scores of the two halves h: rows of the product are keys 16 h + g and 16 h + g + 8,
    // columns query rows 2 c, 2 c + 1
    float s[2][4], t[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[h][j] = t[h][j] = 0.f;
#pragma unroll
    for (int hf = 0; hf < D / 64; ++hf) {
      uint4 ka[2], kb[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ka[h] = *reinterpret_cast<const uint4*>(kst + ka_at<D>(16 * h + g, c + 4 * hf));
        kb[h] = *reinterpret_cast<const uint4*>(kst + ka_at<D>(16 * h + g + 8, c + 4 * hf));
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa = (&ka[h].x)[w], wb = (&kb[h].x)[w];
          const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)wa), a1 = e4m3x2_to_f16x2((uint16_t)wb),
                         a2 = e4m3x2_to_f16x2((uint16_t)(wa >> 16)), a3 = e4m3x2_to_f16x2((uint16_t)(wb >> 16));
          if constexpr (PAIR) {
            mma16816(s[h], a0, a1, a2, a3, qh[4 * hf + w][0], qh[4 * hf + w][1]);
            mma16816(t[h], a0, a1, a2, a3, ql[4 * hf + w][0], ql[4 * hf + w][1]);
          } else {
            mma16816(w & 1 ? t[h] : s[h], a0, a1, a2, a3, qh[4 * hf + w][0], qh[4 * hf + w][1]);
          }
        }
    }
    const bool border = key0 + KA_KEYS > kmin;  // some row does not see some key
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float kf = __shfl_sync(0xffffffffu, ks, 2 * i + h), lv = __shfl_sync(0xffffffffu, lvs, 2 * i + h);
      iv[h] = __shfl_sync(0xffffffffu, ivs, 2 * i + h);
      const float k0 = kf * f0, k1 = kf * f1;
      s[h][0] = fmaf(s[h][0] + t[h][0], k0, lv);
      s[h][1] = fmaf(s[h][1] + t[h][1], k1, lv);
      s[h][2] = fmaf(s[h][2] + t[h][2], k0, lv);
      s[h][3] = fmaf(s[h][3] + t[h][3], k1, lv);
      if (border) {
        const int key = key0 + 16 * h + g;
        if (key >= lim0) s[h][0] = -INFINITY;
        if (key >= lim1) s[h][1] = -INFINITY;
        if (key + 8 >= lim0) s[h][2] = -INFINITY;
        if (key + 8 >= lim1) s[h][3] = -INFINITY;
      }
    }
    // the running maxima grow rarely: rows are reduced and rescaled only then
    float x0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
    float x1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
    if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
      x0 = fmaxf(m0, x0);
      x1 = fmaxf(m1, x1);
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
      }
      const float r0_ = m0 == x0 ? 1.f : ex2(m0 - x0), r1_ = m1 == x1 ? 1.f : ex2(m1 - x1);
      m0 = x0;
      m1 = x1;
      l0 *= r0_;
      l1 *= r1_;
#pragma unroll
      for (int j = 0; j < DG / 2; ++j) {
        o[j][0] *= r0_;
        o[j][1] *= r1_;
        o[j][2] *= r0_;
        o[j][3] *= r1_;
      }
    }
    const float u0 = (m0 == -INFINITY ? 0.f : m0) - KA_LIFT, u1 = (m1 == -INFINITY ? 0.f : m1) - KA_LIFT;
    uint32_t ph[2][2], pl[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float w0 = ex2(s[h][0] - u0), w1 = ex2(s[h][1] - u1), w2 = ex2(s[h][2] - u0), w3 = ex2(s[h][3] - u1);
      l0 = fmaf(w0 + w2, iv[h], l0);
      l1 = fmaf(w1 + w3, iv[h], l1);
      const uint32_t pa = pack_f16(w0, w1), pb = pack_f16(w2, w3);
      ph[h][0] = transpose8x8(pa);
      ph[h][1] = transpose8x8(pb);
      if constexpr (PAIR) {
        const float2 ra = rest_f16(pa, w0, w1), rb = rest_f16(pb, w2, w3);
        pl[h][0] = transpose8x8(pack_f16(ra.x * KA_LOW, ra.y * KA_LOW));
        pl[h][1] = transpose8x8(pack_f16(rb.x * KA_LOW, rb.y * KA_LOW));
      }
    }

    bool nans = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // V: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9, dimensions DG g .. DG g + DG - 1
      uint32_t v[4][VW];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int row = 16 * h + 2 * c + (kk & 1) + 8 * (kk >> 1);
        if constexpr (D == 128) {
          const uint4 u = *reinterpret_cast<const uint4*>(vst + ka_at<D>(row, g));
          v[kk][0] = u.x; v[kk][1] = u.y; v[kk][2] = u.z; v[kk][3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(vst + ka_at<D>(row, g >> 1) + 8 * (g & 1));
          v[kk][0] = u.x; v[kk][1] = u.y;
        }
      }
      if (border) {
        // a NaN code of a key that only some rows see must not reach the others
        // through 0 * NaN: such codes enter the product as 0 and are put back below
        uint32_t bad = 0;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const uint32_t nb = nan_bytes(v[kk][w]);
            bad |= nb;
            v[kk][w] &= ~((nb >> 7) * 0xffu);
          }
        nans |= __any_sync(0xffffffffu, bad != 0);
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // dimensions 4 w + 2 e (rows 0 - 7 of the product) and the next one (rows 8 - 15)
          const uint32_t x = __byte_perm(v[0][w], v[1][w], e ? 0x7362 : 0x5140);
          const uint32_t y = __byte_perm(v[2][w], v[3][w], e ? 0x7362 : 0x5140);
          const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)x), a1 = e4m3x2_to_f16x2((uint16_t)(x >> 16)),
                         a2 = e4m3x2_to_f16x2((uint16_t)y), a3 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
          mma16816(o[2 * w + e], a0, a1, a2, a3, ph[h][0], ph[h][1]);
          if constexpr (PAIR) {
            float low[4];
            mma16816_first(low, a0, a1, a2, a3, pl[h][0], pl[h][1]);
            float(&to)[4] = o[2 * w + e];
            const float2 x = f2_parts(f2_fma(f2(low[0], low[1]), f2(1.0f / KA_LOW, 1.0f / KA_LOW), f2(to[0], to[1])));
            const float2 y = f2_parts(f2_fma(f2(low[2], low[3]), f2(1.0f / KA_LOW, 1.0f / KA_LOW), f2(to[2], to[3])));
            to[0] = x.x; to[1] = x.y; to[2] = y.x; to[3] = y.y;
          }
        }
    }
    if (nans) {
      for (int kk = 0; kk < KA_KEYS; ++kk) {
        const uint8_t* p = vst + ka_at<D>(kk, D == 128 ? g : g >> 1) + (D == 128 ? 0 : 8 * (g & 1));
#pragma unroll
        for (int j = 0; j < DG; ++j) {
          if ((p[j] & 0x7f) != 0x7f) continue;
          if (key0 + kk < lim0) o[j >> 1][(j & 1) * 2] = __int_as_float(0x7fffffff);
          if (key0 + kk < lim1) o[j >> 1][(j & 1) * 2 + 1] = __int_as_float(0x7fffffff);
        }
      }
    }
  }

  // ---- join the warps: rows 2 c and 2 c + 1 of each lane's DG dimensions
#pragma unroll
  for (int d = 4; d < 32; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  cp_async_wait<0>();
  __syncthreads();
  float* ob = reinterpret_cast<float*>(ka_smem);
#pragma unroll
  for (int j = 0; j < DG / 2; ++j) {
    float* p = ob + (warp * KA_ROWS + 2 * c) * C::LD + DG * g + 2 * j;
    *reinterpret_cast<float2*>(p) = make_float2(o[j][0], o[j][2]);
    *reinterpret_cast<float2*>(p + C::LD) = make_float2(o[j][1], o[j][3]);
  }
  if (g == 0) {
    join_m[warp][2 * c] = m0;
    join_m[warp][2 * c + 1] = m1;
    join_l[warp][2 * c] = l0;
    join_l[warp][2 * c + 1] = l1;
  }
  __syncthreads();
  constexpr int PER = KA_ROWS * D / (KA_WARPS * 32);  // output values a thread: 4 or 8
  const int row = tid / (D / PER), d0 = tid % (D / PER) * PER;
  float mt = -INFINITY, lt = 0.f, x[PER];
#pragma unroll
  for (int w = 0; w < KA_WARPS; ++w) mt = fmaxf(mt, join_m[w][row]);
#pragma unroll
  for (int j = 0; j < PER; ++j) x[j] = 0.f;
#pragma unroll
  for (int w = 0; w < KA_WARPS; ++w) {
    const float mw = join_m[w][row], f = mw == mt ? 1.f : ex2(mw - mt);
    lt = fmaf(join_l[w][row], f, lt);
    const float* p = ob + (w * KA_ROWS + row) * C::LD + d0;
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = fmaf(p[j], f, x[j]);
  }
  mt -= KA_LIFT;  // what the sums are relative to
  if (!whole) lt = __int_as_float(0x7fffffff);  // the sequence's length did not fit
  else if (lt == 0.f && limit(r0 + row) > c0) mt = KV_ALL_LOW;
  const auto head_row = [&](int rr) {
    return (int64_t)(first + rr / a.group) * a.heads + kvh * a.group + rr % a.group;
  };
  const auto finish = [&](int rr) {
    lt = kv_whole_sum(mt, lt);
    const bool sees = lt != 0.f;
    const float inv = sees ? 1.0f / lt : 0.f;
    const int64_t rh = head_row(rr);
    T* p = static_cast<T*>(a.out) + rh * D + d0;
#pragma unroll
    for (int j = 0; j < PER; ++j) p[j] = from_f32<T>(sees ? x[j] * inv : 0.f);
    if (a.lse && d0 == 0) a.lse[rh] = sees ? (mt + log2f(lt)) * 0.6931471805599453f : -INFINITY;
  };
  if (a.splits == 1) {
    if (r0 + row < nrows) finish(r0 + row);
    return;
  }
  if (!a.cluster) {
    if (r0 + row >= nrows) return;
    const int64_t rh = head_row(r0 + row);
    float* p = a.part + (rh * a.splits + split) * D + d0;
#pragma unroll
    for (int j = 0; j < PER; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    if (d0 == 0) a.ml[rh * a.splits + split] = make_float2(mt, lt);
    return;
  }
  // the cluster's blocks share out the rows, each reads the others' sums
#pragma unroll
  for (int j = 0; j < PER; ++j) sum_o[row][d0 + j] = x[j];
  if (d0 == 0) sum_ml[row] = make_float2(mt, lt);
  cluster_sync_all();
  const int mine = split + row * a.splits;
  if (mine < KA_ROWS && r0 + mine < nrows) {
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      const float4 v = kv_join_cluster(smem_addr(&sum_ml[mine]), smem_addr(&sum_o[mine][d0 + j]), a.splits, mt, lt);
      x[j] = v.x;
      x[j + 1] = v.y;
      x[j + 2] = v.z;
      x[j + 3] = v.w;
    }
    finish(r0 + mine);
  }
  __syncwarp();
  cluster_sync_all();  // no block leaves while another may still read its sums
}

// Joins the splits of one (row, head).  D / 4 threads cover a split's row, the others take
// other splits at the same time, so that a row split into hundreds of stretches (one
// sequence of 128 Ki tokens) costs a few rounds of loads; each split's weight is worked
// out once.  256 threads for up to 32 splits, 1024 for more (147 splits: the whole call is
// 2.2 us faster with 1024).
constexpr int KJ_MAX = 1024;  // splits whose weights are kept at a time

template <typename T, int D, int KJ_THREADS>
__global__ void __launch_bounds__(KJ_THREADS) kv_attn_join_kernel(const KvBatch b, const int* refused, int heads,
                                                                  const float* part, const float2* ml, int splits,
                                                                  T* out, float* lse) {
  constexpr int COLS = D / 4, LANES = KJ_THREADS / COLS;
  __shared__ float weight[KJ_MAX];
  __shared__ float red[2][KJ_THREADS / 32];
  __shared__ float4 sums[LANES][COLS];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t rh = blockIdx.x;
  const int token = (int)(rh / heads), tid = threadIdx.x, col = tid % COLS, sub = tid / COLS;
  // no sequence's row, or nothing to join: left as it was
  if (b.starts && (*refused || token < b.starts[0] || token >= b.starts[b.seqs])) return;
  const float2* m = ml + rh * splits;
  const float4* p = reinterpret_cast<const float4*>(part + rh * splits * D) + col;
  float mt = -INFINITY, lt = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = tid; s < splits; s += KJ_THREADS) mt = fmaxf(mt, m[s].x);
  mt = warp_max(mt);
  if ((tid & 31) == 0) red[0][tid >> 5] = mt;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KJ_THREADS / 32; ++w) mt = fmaxf(mt, red[0][w]);
  for (int s0 = 0; s0 < splits; s0 += KJ_MAX) {
    const int n = min(KJ_MAX, splits - s0);
    if (s0) __syncthreads();
    for (int s = tid; s < n; s += KJ_THREADS) {
      const float2 v = m[s0 + s];
      const float f = v.x == mt ? 1.f : ex2(v.x - mt);
      // nothing seen there means nothing written to part: no weight, whatever lies there
      weight[s] = v.y == 0.f ? -1.f : f;
      lt += v.y == 0.f ? 0.f : v.y * f;
    }
    __syncthreads();
#pragma unroll 4
    for (int s = sub; s < n; s += LANES) {
      const float f = weight[s];
      if (f < 0.f) continue;
      const float4 v = p[(int64_t)(s0 + s) * COLS];
      x.x = fmaf(v.x, f, x.x);
      x.y = fmaf(v.y, f, x.y);
      x.z = fmaf(v.z, f, x.z);
      x.w = fmaf(v.w, f, x.w);
    }
  }
  lt = warp_sum(lt);
  if ((tid & 31) == 0) red[1][tid >> 5] = lt;
  sums[sub][col] = x;
  __syncthreads();
  if (tid >= COLS) return;
  lt = 0.f;
#pragma unroll
  for (int w = 0; w < KJ_THREADS / 32; ++w) lt += red[1][w];
  lt = kv_whole_sum(mt, lt);
#pragma unroll
  for (int i = 1; i < LANES; ++i) {
    const float4 v = sums[i][col];
    x.x += v.x;
    x.y += v.y;
    x.z += v.z;
    x.w += v.w;
  }
  const bool sees = lt != 0.f;
  const float inv = sees ? 1.0f / lt : 0.f;
  T* o = out + rh * D + 4 * col;
  o[0] = from_f32<T>(sees ? x.x * inv : 0.f);
  o[1] = from_f32<T>(sees ? x.y * inv : 0.f);
  o[2] = from_f32<T>(sees ? x.z * inv : 0.f);
  o[3] = from_f32<T>(sees ? x.w * inv : 0.f);
  if (lse && tid == 0) lse[rh] = sees ? (mt + log2f(lt)) * 0.6931471805599453f : -INFINITY;
}

// ------------------------------------------------------------------- host
struct KvAttnPlan {
  int tile_rows;  // 128 (kv_attention_tile.cu), 256 (kv_attention_wide.cu) or 0: 8 rows a block
  int64_t items;
  int per_seq, chunk, splits;
  bool cluster;
  int64_t whole, tails;  // 256-row tiles: items that are one block, items of `splits` blocks
  int64_t workspace;     // bytes
};

static int64_t kv_attn_items(const rtr_kv_batch* b, int group, int shift, int& per_seq) {
  if (b->starts) {
    per_seq = 0;
    return ((int64_t)b->rows * group >> shift) + b->seqs;
  }
  per_seq = (int)(((int64_t)(b->rows / b->seqs) * group + (1 << shift) - 1) >> shift);
  return (int64_t)per_seq * b->seqs;
}

// Of the tiles that a ragged call may have (a sequence's last one is half full on average),
// as many as it will hardly exceed: planned for the most there can be, 5 sequences of 3,000 - 6,000 keys with 33 -
// 135 rows take 31.1 us instead of 27.9.
static int64_t kv_likely_items(const rtr_kv_batch* b, int group, int shift, int64_t items) {
  if (!b->starts) return items;
  const double mean = (double)b->rows * group / (1 << shift) + 0.5 * b->seqs;
  return std::min(items, std::max((int64_t)b->seqs, (int64_t)std::ceil(mean + std::sqrt(b->seqs / 12.0))));
}

// Tiles of 8 rows: stretches and the time to expect, in ns.
static KvAttnPlan kv_plan_rows(const rtr_kv_cache* c, const rtr_kv_batch* b, int group, bool f32, int sms, int64_t& ns) {
  KvAttnPlan p = {};
  p.items = kv_attn_items(b, group, 3, p.per_seq);
  const int64_t most = (int64_t)b->table_width * c->page, base = p.items * c->kv_heads;
  // A stretch has at least 512 keys: below that a block is bound by the latency of
  // finding its pages, and joining costs more than it saves (61 sequences of 30 - 300
  // keys, 14 heads: 5.5 us in one stretch, 5.8 in three); at most 1024, which a warp's lanes
  // can hold the pages of and at which ragged batches spread (24 sequences of 6,000 -
  // 32,000 keys: 89.8 us, with 512 100.5); between them as many as give two blocks an SM (one
  // sequence of 128 Ki keys: 19.1 us, with three an SM 19.0, with 512 keys 23.0).
  const int64_t want = 2 * (int64_t)sms;
  int64_t chunk = base >= want ? most : most * base / want;
  chunk = (chunk + 63) / 64 * 64;
  if (chunk < 512) chunk = 512;
  if (chunk > KA_MAX_CHUNK) chunk = KA_MAX_CHUNK;
  p.chunk = (int)chunk;
  p.splits = (int)((most + chunk - 1) / chunk);
  p.cluster = p.splits > 1 && p.splits <= KV_CLUSTER;
  // measured: 8 rows x 18,500 (fp32 16,000) keys a us at head_dim 128, 45,000 (35,000) at 64
  const int64_t rate = c->head_dim == 128 ? (f32 ? 16000 : 18500) : f32 ? 35000 : 45000;
  ns = 5000 + base * most * 1000 / rate + (p.splits > 1 ? 3000 : 0);
  return p;
}

// What a block of 128 rows needs for 128 keys.
static int kv_tile_ns(const rtr_kv_cache* c, bool f32) {
  return c->head_dim == 128 ? (f32 ? 1700 : 1100) : f32 ? 1350 : 1150;
}

// Tiles of 128 rows.
static KvAttnPlan kv_plan_tiles(const rtr_kv_cache* c, const rtr_kv_batch* b, int group, bool f32, int sms, int64_t& ns) {
  KvAttnPlan p = {};
  p.tile_rows = KT_ROWS;
  p.items = kv_attn_items(b, group, 7, p.per_seq);
  const int64_t base = kv_likely_items(b, group, 7, p.items) * c->kv_heads;
  const int64_t all = ((int64_t)b->table_width * c->page + KT_KEYS - 1) / KT_KEYS;
  // A block costs its key tiles and about six more (q, first and last tile, output), a
  // cluster's join three, a join through memory eight.  Clusters of three and more fill
  // about six of seven SMs.
  int64_t best = INT64_MAX;
  for (int64_t s = (all * KT_KEYS + KT_MAX_CHUNK - 1) / KT_MAX_CHUNK, end = s + 63; s <= end && s <= all; ++s) {
    const int64_t per = (all + s - 1) / s, splits = (all + per - 1) / per;
    const int64_t wave = splits >= 3 && splits <= KV_CLUSTER ? sms * 6 / 7 : sms;
    const int64_t cost = (base * splits + wave - 1) / wave * (per + 6) + (splits == 1 ? 0 : splits <= KV_CLUSTER ? 3 : 8);
    if (cost < best) {
      best = cost;
      p.chunk = (int)(per * KT_KEYS);
      p.splits = (int)splits;
    }
  }
  p.cluster = p.splits > 1 && p.splits <= KV_CLUSTER;
  ns = best * kv_tile_ns(c, f32);
  return p;
}

// What a block of 256 rows needs for 128 keys, and for its start and end in these units.
constexpr int KW_TILE_NS = 1750, KW_BLOCK = 7;

// Tiles of 256 rows.  Items that fill all SMs are blocks of their own; what is left is split
// along its keys, so that the last wave is a short one, and joined through memory.
static KvAttnPlan kv_plan_wide(const rtr_kv_cache* c, const rtr_kv_batch* b, int group, int sms, int64_t& ns) {
  KvAttnPlan p = {};
  p.tile_rows = KW_ROWS;
  p.items = kv_attn_items(b, group, 8, p.per_seq);
  const int64_t base = p.items * c->kv_heads;
  const int64_t all = ((int64_t)b->table_width * c->page + KT_KEYS - 1) / KT_KEYS, most = KW_MAX_CHUNK / KT_KEYS;
  const int64_t waves = all > most ? 0 : base / sms;
  int64_t best = INT64_MAX;
  for (int64_t s = (all + most - 1) / most, end = s + 63; s <= end && s <= all; ++s) {
    const int64_t per = (all + s - 1) / s, splits = (all + per - 1) / per, left = base - waves * sms;
    const int64_t cost = waves * (all + KW_BLOCK) + (left * splits + sms - 1) / sms * (per + KW_BLOCK) + (splits == 1 ? 0 : 3);
    if (cost < best) {
      best = cost;
      p.whole = splits == 1 ? base : waves * sms;
      p.chunk = (int)(per * KT_KEYS);
      p.splits = (int)splits;
    }
  }
  p.tails = base - p.whole;
  ns = best * KW_TILE_NS;
  return p;
}

// The kernel whose expected time is less.  Measured, 28 / 4 heads of 128, bf16, tiles of
// 128 against tiles of 8 rows: 8 sequences of 1,200 keys with 2 new tokens 13.2 : 10.8 us,
// 4 13.4 : 12.3, 16 15.1 : 36.6; one of 300 keys with 64 11.5 : 8.0 us, with 256 11.3 : 15.0.
// Tiles of 256 against 128: 32 sequences of 4,096 keys with 64 157 : 199 us, 4 of 512 keys with
// 256 21 : 24.6, one of 4,096 with 1,024 77 : 91, with 512 52 : 49.
static KvAttnPlan kv_attn_plan(const rtr_kv_cache* c, const rtr_kv_batch* b, int heads, bool f32, int sms) {
  const int group = heads / c->kv_heads;
  int64_t rows_ns, tiles_ns;
  KvAttnPlan p = kv_plan_rows(c, b, group, f32, sms, rows_ns);
  if (rows_ns > 7 * kv_tile_ns(c, f32)) {  // what one key tile costs at least
    const KvAttnPlan tiles = kv_plan_tiles(c, b, group, f32, sms, tiles_ns);
    if (tiles_ns < rows_ns) {
      p = tiles;
      if (!f32 && c->head_dim == 128) {
        int64_t wide_ns;
        const KvAttnPlan wide = kv_plan_wide(c, b, group, sms, wide_ns);
        if (wide_ns < tiles_ns && wide.whole + wide.tails * wide.splits <= INT32_MAX / KW_ROWS) p = wide;
      }
    }
  }
  if (p.tile_rows == KW_ROWS)
    p.workspace = p.tails * KW_ROWS * (p.splits * (int64_t)(c->head_dim * 4 + 8) + 4);
  else  // with starts one row more: KvAttn::refused lies behind the sums
    p.workspace = p.splits > 1 && !p.cluster
                      ? ((int64_t)b->rows * heads * p.splits + (b->starts != nullptr)) * (c->head_dim * 4 + 8) : 0;
  return p;
}

// What rtr_debug_wait_control has set, by device.
constexpr int KV_DEVICES = 64;
struct KvWait {
  std::atomic<long long> cycles{kWaitCycles};
  std::atomic<int> withhold{0};
};
static KvWait kv_wait[KV_DEVICES];
void kv_attn_wait_control(int device, long long wait_cycles, int withhold) {
  if (device < 0 || device >= KV_DEVICES) return;
  kv_wait[device].cycles.store(wait_cycles, std::memory_order_relaxed);
  kv_wait[device].withhold.store(withhold, std::memory_order_relaxed);
}

static const char* kv_attn_check(const rtr_kv_cache* c, const rtr_kv_batch* b, int heads) {
  if (const char* e = kv_check(c, b)) return e;
  if (heads < 1 || heads % c->kv_heads) return "heads must be a multiple of kv_heads";
  if (heads > 16384) return "at most 16384 heads";
  if ((int64_t)b->rows * heads > INT32_MAX) return "at most 2^31 - 1 rows x heads in one call";
  return nullptr;
}

template <typename T, int D> static cudaError_t kv_attn_launch(const KvAttn& a, const KvAttnPlan& p, int device, cudaStream_t st) {
  cudaError_t e;
  if (p.tile_rows == KW_ROWS) {
    const int64_t rows = p.tails * KW_ROWS * p.splits;
    KvAttn w = a;
    w.ml = reinterpret_cast<float2*>(a.part + rows * D);
    return kv_attn_wide(w, KwShare{(int)p.whole, (int)p.tails, reinterpret_cast<int*>(w.ml + rows)}, device, st);
  }
  if (p.tile_rows) {
    e = kv_attn_tile(a, p.items, std::is_same<T, float>::value, device, st);
  } else {
    static std::atomic<uint64_t> done;
    e = kv_allow_smem(kv_attn_rows_kernel<T, D>, KaCfg<D>::SMEM, done, device);
    if (e != cudaSuccess) return e;
    e = kv_launch(kv_attn_rows_kernel<T, D>, dim3((unsigned)p.items, a.c.kv_heads, a.splits), KA_WARPS * 32,
                  KaCfg<D>::SMEM, a.cluster ? a.splits : 1, st, a);
  }
  if (e != cudaSuccess || a.splits == 1 || a.cluster) return e;
  const auto join = [&](auto kernel, int threads) {
    return launch_pdl(PDL_ATTN, kernel, dim3((unsigned)(a.b.rows * a.heads)), dim3(threads), 0, st, a.b,
                      (const int*)a.refused, a.heads, (const float*)a.part, (const float2*)a.ml, a.splits,
                      static_cast<T*>(a.out), a.lse);
  };
  return a.splits <= 32 ? join(kv_attn_join_kernel<T, D, 256>, 256) : join(kv_attn_join_kernel<T, D, 1024>, 1024);
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_kv_attention_workspace(const rtr_kv_cache* cache, const rtr_kv_batch* batch, int32_t dtype, int32_t heads,
                               int32_t device, int64_t* bytes) {
  if (!bytes) return set_error(RTR_ERR_ARG, "null bytes");
  if (const char* e = kv_attn_check(cache, batch, heads)) return set_error(RTR_ERR_ARG, e);
  *bytes = 0;
  if (!batch->rows) return RTR_OK;
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  *bytes = kv_attn_plan(cache, batch, heads, dtype == RTR_DTYPE_F32, on.sms).workspace;
  return RTR_OK;
}

int rtr_kv_attention(const rtr_kv_cache* cache, const rtr_kv_batch* batch, const void* q_dev, int32_t dtype,
                     int32_t heads, int64_t q_token_stride, int32_t causal, float scale, void* out_dev, float* lse_dev,
                     void* workspace_dev, int64_t workspace_bytes, int32_t device, void* stream) {
  if (const char* e = kv_attn_check(cache, batch, heads)) return set_error(RTR_ERR_ARG, e);
  if (!batch->rows) return RTR_OK;
  if (dtype != RTR_DTYPE_F32 && dtype != RTR_DTYPE_BF16)
    return set_error(RTR_ERR_ARG, "dtype must be float32 or bfloat16");
  const int size = dtype == RTR_DTYPE_F32 ? 4 : 2;
  if (!q_dev || !out_dev) return set_error(RTR_ERR_ARG, "null q or out");
  if ((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev) | (uintptr_t)(q_token_stride * size)) & 15)
    return set_error(RTR_ERR_ARG, "q, its stride and out must be multiples of 16 bytes");
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  const KvAttnPlan p = kv_attn_plan(cache, batch, heads, dtype == RTR_DTYPE_F32, on.sms);
  if (p.items > INT32_MAX || p.splits > 65535 || cache->kv_heads > 65535)
    return set_error(RTR_ERR_ARG, "too many rows or keys for one call");
  if (p.workspace && (!workspace_dev || workspace_bytes < p.workspace || (reinterpret_cast<uintptr_t>(workspace_dev) & 15)))
    return set_error(RTR_ERR_ARG, "workspace missing, too small or not aligned to 16 bytes");
  KvAttn a;
  a.c = kv_device_cache(cache);
  a.b = kv_device_batch(batch);
  a.q = q_dev;
  a.q_token = q_token_stride;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.group_inverse = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  a.causal = causal != 0;
  a.factor = scale * 1.4426950408889634f;
  a.out = out_dev;
  a.lse = lse_dev;
  a.part = static_cast<float*>(workspace_dev);
  a.ml = reinterpret_cast<float2*>(a.part + (int64_t)batch->rows * heads * p.splits * cache->head_dim);
  a.refused = batch->starts && p.splits > 1 && !p.cluster && p.tile_rows != KW_ROWS
                  ? reinterpret_cast<int*>(a.ml + (int64_t)batch->rows * heads * p.splits) : nullptr;
  a.per_seq = p.per_seq;
  a.chunk = p.chunk;
  a.splits = p.splits;
  a.cluster = p.cluster;
  const KvWait& w = kv_wait[device >= 0 && device < KV_DEVICES ? device : 0];
  a.wait_cycles = w.cycles.load(std::memory_order_relaxed);
  a.withhold = w.withhold.load(std::memory_order_relaxed);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == RTR_DTYPE_F32)
    e = cache->head_dim == 128 ? kv_attn_launch<float, 128>(a, p, device, st) : kv_attn_launch<float, 64>(a, p, device, st);
  else
    e = cache->head_dim == 128 ? kv_attn_launch<__nv_bfloat16, 128>(a, p, device, st)
                               : kv_attn_launch<__nv_bfloat16, 64>(a, p, device, st);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
