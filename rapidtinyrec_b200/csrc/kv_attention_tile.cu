// Attention over the 8-bit KV cache for many query rows: tiles of 128 (token,
// head of the group) rows of one KV head on the 5th-generation tensor cores.
//
// The mathematics is that of kv_attention.cu: scores of the codes as they are, one
// running maximum of score + log2(V scale) a row.  A block walks its keys in tiles of
// 128; per tile S = Q K^T and O = P V are tcgen05 products with fp32 accumulators in
// tensor memory.  Warps have one role each:
//   rows     8 warps: scores to weights, which they write over the scores as the A
//            operand of P V;
//   codes    read K and V of the next tiles from the pages into registers, turn them
//            into fp16 and store them as swizzled operands, V transposed;
//   products one thread issues the products.
// There are two buffers of K, V, S and O, tile i in buffer i % 2.
//
// bf16 rows: two threads a row, each with 64 of a tile's keys, its own maximum, sum and
// O in tensor memory; the two are joined at the end.  Weights are computed in one pass with
// the maximum as it stands; only where a score exceeds it by more than 2^KT_SLACK (weights stay
// below 2^15) are O and the sum rescaled and the pass repeated.
// fp32 rows: q and the weights enter as fp16 pairs, two products each.  The tensor core's
// own accumulation drifts over thousands of keys, so tensor memory sums one tile only: two
// threads a row (64 scores of the tile each) add it to half of the output's dimensions in
// registers, by IEEE operations.  Weights are relative to their own tile's maximum, which the
// addition makes up for: the low parts of a pair keep 22 bits down to 2^-17 of the largest
// weight of 128 keys (tensor memory has no room for a product of their own), whatever other
// tiles hold.
//
// What bounds it is the chain of a tile, weights - O - S (about 2,600 cycles for 128 keys at
// head_dim 128, of which exponentials need 1,024 and products 1,024).  2 x 1,024 rows at the end of
// 6,000 keys: 28 / 4 heads of 128, bf16, 248 us (650 TFLOP/s of what the mask leaves;
// kv_attention_wide.cu 192); 12 / 2, fp32, 154 us (448); 14 / 2 of 64 101 (399, bf16) and 153 us
// (263, fp32).  50 beams over 719 keys, 28 / 4, 11.5 us.
#include <cuda_runtime.h>

#include <type_traits>

#include "engine.h"
#include "kv_attention_tile.cuh"
#include "kv_host.h"

namespace rtr {

template <int D, bool PAIR> struct KtCfg {
  // row threads need 128 registers, which leaves room for four code warps; eight, with 96
  // registers, were no faster
  static constexpr int CODE_WARPS = 4;
  static constexpr int CODE_THREADS = 32 * CODE_WARPS;
  static constexpr int THREADS = KT_ROW_THREADS + CODE_THREADS + 32;
  static constexpr int P_ARRIVALS = PAIR ? 256 : 128;          // row threads of a tile
  static constexpr int PANELS = D / 64;                        // 128-byte panels of a q or k row
  static constexpr int Q_PLANE = PANELS * KT_ROWS * 128;
  static constexpr int Q_BYTES = (PAIR ? 2 : 1) * Q_PLANE;
  static constexpr int K_BYTES = PANELS * KT_KEYS * 128;       // [panel][key][64 dims]
  static constexpr int V_BYTES = 2 * D * 128;                  // [64 keys][dim][64 keys]: V transposed
  static constexpr int Q_OFF = 0, K_OFF = Q_BYTES, V_OFF = K_OFF + 2 * K_BYTES;
  static constexpr int SEG_OFF = V_OFF + 2 * V_BYTES;          // int64 offsets, then 3 floats a segment
  static constexpr int ROW_OFF = SEG_OFF + KT_SEGS * 20;       // per row: row of out, keys it sees
  static constexpr int RED_OFF = ROW_OFF + KT_ROWS * 8;        // [2][2][128] maxima
  static constexpr int BAR_OFF = RED_OFF + 2 * 2 * KT_ROWS * 4;
  // the finished tile (rows of STAGE_LD floats) lies over the last operands, what a cluster's
  // blocks send each other over the first
  static constexpr int STAGE_LD = D + 4;
  static constexpr int STAGE_OFF = SEG_OFF - KT_ROWS * STAGE_LD * 4;
  static constexpr int RECV_ROWS = KT_ROWS + KV_CLUSTER;       // ceil(128 / splits) rows from each block
  static_assert(RECV_ROWS * D * 4 + RECV_ROWS * 8 <= STAGE_OFF, "both lie over the operands");
  static constexpr int SMEM = BAR_OFF + 256 + 1024;            // 1024: alignment of the operands
};

struct KtBars {
  uint64_t q_full, k_full[2], v_full[2], s_full[2], p_full[2][2], o_full[2][2], o_free[2];  // p, o: [half][buffer]
  uint32_t tmem;
  int abort_flag;
  int nans;  // V has NaN codes in a tile that not every row sees as a whole
};
static_assert(sizeof(KtBars) <= 256, "barriers fit their part of shared memory");

RTR_DEVICE void st_cluster_f4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
RTR_DEVICE void st_cluster_f2(uint32_t addr, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(KtCfg<D, std::is_same<T, float>::value>::THREADS, 1) kv_attn_tile_kernel(const KvAttn a) {
  constexpr bool PAIR = std::is_same<T, float>::value;
  using C = KtCfg<D, PAIR>;
  constexpr float LIFT = PAIR ? KA_LIFT : KT_LIFT;
  constexpr int HD = D / 2;    // dimensions of the output a row thread finishes
  constexpr int NL = D / 8;    // of those, the ones with the same d % 4
  extern __shared__ uint8_t kt_smem_raw[];
  __shared__ int slot[2];
  uint8_t* smem = kt_smem_raw + ((1024u - (smem_addr(kt_smem_raw) & 1023u)) & 1023u);
  uint8_t* qs = smem + C::Q_OFF;
  int64_t* seg_at = reinterpret_cast<int64_t*>(smem + C::SEG_OFF);
  float* seg_k = reinterpret_cast<float*>(seg_at + KT_SEGS);
  float* seg_lv = seg_k + KT_SEGS;
  float* seg_iv = seg_lv + KT_SEGS;
  int* row_out = reinterpret_cast<int*>(smem + C::ROW_OFF);
  int* row_lim = row_out + KT_ROWS;
  float* red = reinterpret_cast<float*>(smem + C::RED_OFF);
  KtBars& bars = *reinterpret_cast<KtBars*>(smem + C::BAR_OFF);
  volatile int* abort_flag = &bars.abort_flag;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int kvh = blockIdx.y, split = blockIdx.z;
  pdl_launch_dependents();
  pdl_wait();

  int seq;
  int64_t item0;
  if (a.b.starts) {
    seq = kv_find_seq(a.b, blockIdx.x, a.group, 7, 1, a.c.status, slot, item0);
    if (a.refused && tid == 0) *a.refused = seq == -2;  // every block says the same
    if (seq < 0) return;
  } else {
    seq = (int)blockIdx.x / a.per_seq;
    item0 = (int64_t)seq * a.per_seq;
  }
  // What needs no other load's result is loaded first: the length, the code warps' page
  // numbers and the row warps' q.
  int first, count, len = a.b.lens[seq];
  if (!kv_rows(a.b, seq, a.c.status, first, count)) return;
  const int nrows = count * a.group, r0 = (int)(blockIdx.x - item0) * KT_ROWS;
  if (r0 >= nrows) return;
  const int rows = min(KT_ROWS, nrows - r0), c0 = split * a.chunk;
  constexpr int QPER = 16 / sizeof(T), QLPR = D / QPER, QRPI = 32 / QLPR;  // q: values of 16 bytes, lanes of a row, rows of a load
  constexpr int QLOADS = 16 / QRPI, QSTEP = QLOADS < 8 ? QLOADS : 8;
  uint4 q0[QSTEP];
  const int token0 = r0 / a.group, head0 = r0 - token0 * a.group;  // of the tile's first row
  // token and head (of the group) of a row of the tile
  const auto place = [&](int row, int& token, int& head) {
    const int t = kv_div(a, head0 + min(row, rows - 1));
    token = token0 + t;
    head = head0 + min(row, rows - 1) - t * a.group;
  };
  const auto load_q = [&](int base, uint4 (&u)[QSTEP]) {
#pragma unroll
    for (int j = 0; j < QSTEP; ++j) {
      const int row = warp * 16 + (base + j) * QRPI + lane / QLPR;
      int token, head;
      place(row, token, head);
      const T* p = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.q_token +
                   (kvh * a.group + head) * D + (lane % QLPR) * QPER;
      u[j] = row < rows ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  if (warp < 8) load_q(0, q0);
  const bool whole = kv_len_fits(a.c, a.b, len, 0);
  if (!whole) len = 0;  // the sequence's rows become NaN
  // keys that a row of the tile sees; of all rows, the least and the most
  const auto limit = [&](int row) { return a.causal ? max(0, len - count + token0 + kv_div(a, head0 + min(row, rows - 1)) + 1) : len; };
  const int kmin = limit(0), kmax = limit(rows - 1), c1 = c0 + min(kmax - c0, a.chunk);
  if (c1 <= c0 && split > 0 && !a.cluster) {  // a stretch behind the last key (the first one reports rows that see nothing)
    if (tid < rows) {
      const int token = (r0 + tid) / a.group;
      const int64_t rh = (int64_t)(first + token) * a.heads + kvh * a.group + (r0 + tid - token * a.group);
      a.ml[rh * a.splits + split] = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  const int n = c1 > c0 ? (c1 - c0 + KT_KEYS - 1) / KT_KEYS : 0;
  const int segs = c1 > c0 ? (c1 - c0 + 15) / 16 : 0;  // 16-key segments of the stretch

  if (tid == 0) {
    mbar_init(smem_addr(&bars.q_full), KT_ROW_THREADS);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&bars.k_full[i]), C::CODE_THREADS);
      mbar_init(smem_addr(&bars.v_full[i]), C::CODE_THREADS);
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_addr(&bars.p_full[h][i]), C::P_ARRIVALS);
        mbar_init(smem_addr(&bars.o_full[h][i]), 1);
      }
      mbar_init(smem_addr(&bars.o_free[i]), KT_ROW_THREADS);
      mbar_init(smem_addr(&bars.s_full[i]), 1);
    }
    bars.nans = 0;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 + C::CODE_WARPS) tmem_alloc(smem_addr(&bars.tmem), 512);
  if (tid < KT_ROWS) {
    int token, head;
    place(tid, token, head);
    row_out[tid] = (first + token) * a.heads + kvh * a.group + head;
    row_lim[tid] = limit(tid);
  }
  if (tid >= KT_ROW_THREADS)
    kt_segments(a, seq, kvh, c0, segs, tid - KT_ROW_THREADS, C::THREADS - KT_ROW_THREADS, seg_at, seg_k, seg_lv, seg_iv);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(bars.tmem);
  constexpr uint32_t S_COLS = KT_KEYS, O_AT = 2 * S_COLS;

  if (warp < 8) {
    // ------------------------------------------------------------- rows
    const int half = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    {
      // q as fp16 (pairs), each row times a power of two; a warp takes 16 rows
      constexpr int PER = QPER, LPR = QLPR, RPI = QRPI, LOADS = QLOADS, STEP = QSTEP;
      const int sub = lane / LPR, col = lane % LPR, unit = col * PER / 8;
      uint4 u[STEP];
#pragma unroll
      for (int base = 0; base < LOADS; base += STEP) {
        if (base == 0) {
#pragma unroll
          for (int j = 0; j < STEP; ++j) u[j] = q0[j];
        } else {
          load_q(base, u);
        }
        uint32_t top[STEP];  // magnitudes order as their bits do
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
          const uint32_t m = PAIR ? 0x7fffffffu : 0x7fff7fffu, w[4] = {u[j].x & m, u[j].y & m, u[j].z & m, u[j].w & m};
          if constexpr (PAIR) {
            top[j] = max(max(w[0], w[1]), max(w[2], w[3]));
          } else {
            const uint32_t t = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
            top[j] = max(t << 16, t & 0xffff0000u);
          }
        }
        if constexpr (LPR == 32) {
#pragma unroll
          for (int j = 0; j < STEP; ++j) top[j] = __reduce_max_sync(0xffffffffu, top[j]);
        } else {
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1)
#pragma unroll
            for (int j = 0; j < STEP; ++j) top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
        }
        // the row's place in the operand: RPI rows on, 128 RPI bytes on and other swizzle bits
        uint8_t* const at = qs + (unit >> 3) * KT_ROWS * 128 + (warp * 16 + base * RPI + sub) * 128 + (PAIR ? 8 * (col & 1) : 0);
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
          const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
          float x[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            if constexpr (PAIR) x[i] = __uint_as_float(w[i]);
            else x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
          }
          const int e = kv_row_exponent(__uint_as_float(top[j]));
          const float up = copysignf(kv_pow2(-e), a.factor);  // the factor back stays positive: see below
          if (col == 0) red[warp * 16 + (base + j) * RPI + sub] = kv_pow2(e) * fabsf(a.factor);
          uint32_t hi[PER / 2], lo[PER / 2];
#pragma unroll
          for (int i = 0; i < PER / 2; ++i) {
            hi[i] = pack_f16(x[2 * i] * up, x[2 * i + 1] * up);
            const float2 b = rest_f16(hi[i], x[2 * i] * up, x[2 * i + 1] * up);
            lo[i] = pack_f16(b.x, b.y);
          }
          uint8_t* to = at + j * RPI * 128 + ((((unit & 7) ^ sub) ^ ((base + j) * RPI & 7)) << 4);
          if constexpr (PAIR) {
            *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(to + C::Q_PLANE) = make_uint2(lo[0], lo[1]);
          } else {
            *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          }
        }
      }
      fence_proxy_async();
      mbar_arrive(smem_addr(&bars.q_full));
    }
    row_barrier();
    const float f = red[r];  // back to the score, in units of log2; positive
    row_barrier();
    const int lim = row_lim[r];
    uint64_t o[HD / 2];  // pairs; value t * NL + l: dimension half * HD + 4 l + t
    float m = -INFINITY, l = 0.f;

    if constexpr (PAIR) {
#pragma unroll
      for (int i = 0; i < HD / 2; ++i) o[i] = 0;
      float keep = 1.f, take = 1.f;  // factors of what was summed before the last tile, and of that tile

      // adds the finished product of tile i, whose weights are relative to that tile's maximum
      const auto add_product = [&](int i, float keep_, float take_) {
        mbar_wait(smem_addr(&bars.o_full[0][i & 1]), (i >> 1) & 1, abort_flag, a.wait_cycles);
        tc_fence_after();
        const uint32_t at = tmem + lanes + O_AT + (i & 1) * 128 + half * NL;
        const uint64_t old2 = f2(keep_, keep_), new2 = f2(take_, take_);
        uint32_t v[2][NL];
        tmem_ld_cols(at, v[0]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          tmem_ld_wait();
          if (t < 3) tmem_ld_cols(at + (t + 1) * (D / 4), v[(t + 1) & 1]);
#pragma unroll
          for (int j = 0; j < NL / 2; ++j)
            o[t * NL / 2 + j] = f2_fma(f2(v[t & 1][2 * j], v[t & 1][2 * j + 1]), new2, f2_mul(o[t * NL / 2 + j], old2));
        }
        tc_fence_before();
        mbar_arrive(smem_addr(&bars.o_free[i & 1]));
      };

      for (int i = 0; i < n; ++i) {
        mbar_wait(smem_addr(&bars.s_full[i & 1]), (i >> 1) & 1, abort_flag, a.wait_cycles);
        tc_fence_after();
        const uint32_t st = tmem + lanes + (i & 1) * S_COLS + half * 64;
        const int key0 = c0 + i * KT_KEYS + half * 64, seg0 = i * 8 + half * 4;
        const bool border = key0 + 64 > kmin;
        float mx = -INFINITY;
        uint32_t v[2][16];
        tmem_ld16(st, v[0]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int s = min(seg0 + g, segs - 1);
          const float kf = f * seg_k[s], lv = seg_lv[s];
          tmem_ld_wait();
          if (g < 3) tmem_ld16(st + 16 * (g + 1), v[(g + 1) & 1]);
          float top = -INFINITY;
          if (border) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (key0 + 16 * g + j < lim) top = fmaxf(top, __uint_as_float(v[g & 1][j]));
          } else {
#pragma unroll
            for (int j = 0; j < 16; j += 2)
              top = fmaxf(top, fmaxf(__uint_as_float(v[g & 1][j]), __uint_as_float(v[g & 1][j + 1])));
          }
          // kf is positive: the largest product of a segment gives its largest score
          mx = fmaxf(mx, top == -INFINITY ? top : fmaf(top, kf, lv));
        }
        float* rm = red + (i & 1) * 2 * KT_ROWS;
        rm[half * KT_ROWS + r] = mx;
        halves_barrier(warp & 3);
        const float top = fmaxf(rm[r], rm[KT_ROWS + r]), all = fmaxf(m, top);
        const float kept = keep, took = take;  // of the tile before
        keep = m == all ? 1.f : ex2(m - all);
        take = top == all ? 1.f : ex2(top - all);
        m = all;
        float part_l = 0.f;
        const float u = (top == -INFINITY ? 0.f : top) - LIFT;
        // 16 keys at a time, the next ones on their way: few registers are left beside o
        tmem_ld16(st, v[0]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int s = min(seg0 + g, segs - 1);
          const float kf = f * seg_k[s], lv = seg_lv[s] - u, iv = seg_iv[s];
          const uint64_t kf2 = f2(kf, kf), lv2 = f2(lv, lv);
          tmem_ld_wait();
          if (g < 3) tmem_ld16(st + 16 * (g + 1), v[(g + 1) & 1]);
          uint64_t sums = 0;
          uint32_t w[PAIR ? 16 : 8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float2 x = f2_parts(f2_fma(f2(v[g & 1][2 * j], v[g & 1][2 * j + 1]), kf2, lv2));
            if (border) {
              if (key0 + 16 * g + 2 * j >= lim) x.x = -INFINITY;
              if (key0 + 16 * g + 2 * j + 1 >= lim) x.y = -INFINITY;
            }
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sums = f2_add(sums, f2(x.x, x.y));
            w[j] = pack_f16(x.x, x.y);
            if constexpr (PAIR) {
              const float2 b = rest_f16(w[j], x.x, x.y);
              w[8 + j] = pack_f16(b.x, b.y);
            }
          }
          const float sum = f2_parts(sums).x + f2_parts(sums).y;
          part_l = fmaf(sum, iv, part_l);
          tmem_st_words(st + 16 * g, w);  // over the scores just read
        }
        l = fmaf(part_l, take, l * keep);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_addr(&bars.p_full[0][i & 1]));
        if (i > 0) add_product(i - 1, kept, took);
      }
      if (n > 0) add_product(n - 1, keep, take);
      // the row's two halves of the sum
      halves_barrier(warp & 3);
      red[half * KT_ROWS + r] = l;
      halves_barrier(warp & 3);
      l = red[r] + red[KT_ROWS + r];
    } else {
      const uint32_t ot = tmem + lanes + O_AT + half * 128;
      for (int i = 0; i < n; ++i) {
        mbar_wait(smem_addr(&bars.s_full[i & 1]), (i >> 1) & 1, abort_flag, a.wait_cycles);
        tc_fence_after();
        const uint32_t st = tmem + lanes + (i & 1) * S_COLS + half * 64;
        const int key0 = c0 + i * KT_KEYS + half * 64, seg0 = i * 8 + half * 4;
        const bool border = key0 + 64 > kmin;
        // One pass with the maximum as it stands, which also finds the tile's own; where
        // that is too far above, a second one with the new maximum.
        uint32_t w[32];
        float mx, part_l;
        const auto weigh_keys = [&](float u, auto at_border) {
          constexpr bool BORDER = decltype(at_border)::value;
          uint32_t v[2][16];
          tmem_ld16(st, v[0]);
          mx = -INFINITY;
          part_l = 0.f;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int s = min(seg0 + g, segs - 1);
            const float kf = f * seg_k[s], lv = seg_lv[s], iv = seg_iv[s];
            const uint64_t kf2 = f2(kf, kf), lv2 = f2(lv - u, lv - u);
            tmem_ld_wait();
            uint32_t(&x)[16] = v[g & 1];
            if (g < 3) tmem_ld16(st + 16 * (g + 1), v[(g + 1) & 1]);
            float top = -INFINITY;
            uint64_t sums = 0;
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              float z[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                z[e] = BORDER && key0 + 16 * g + j + e >= lim ? -INFINITY : __uint_as_float(x[j + e]);
              top = fmaxf(top, fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                float2 y = f2_parts(f2_fma(f2(x[j + e], x[j + e + 1]), kf2, lv2));
                if constexpr (BORDER) {  // after the product: the scales of a page that the row does not see may be anything
                  if (key0 + 16 * g + j + e >= lim) y.x = -INFINITY;
                  if (key0 + 16 * g + j + e + 1 >= lim) y.y = -INFINITY;
                }
                y.x = ex2(y.x);
                y.y = ex2(y.y);
                sums = f2_add(sums, f2(y.x, y.y));
                w[8 * g + (j + e) / 2] = pack_f16(y.x, y.y);
              }
            }
            part_l = fmaf(f2_parts(sums).x + f2_parts(sums).y, iv, part_l);
            // the factors are positive: the largest product of a segment gives its largest score
            mx = fmaxf(mx, top == -INFINITY ? top : fmaf(top, kf, lv));
          }
        };
        const auto weigh = [&] {
          const float u = (m == -INFINITY ? 0.f : m) - LIFT;
          if (border) weigh_keys(u, std::true_type{});
          else weigh_keys(u, std::false_type{});
        };
        if (i == 0) {
          // nothing to go by: the maximum alone first
          uint32_t v[2][32];
          tmem_ld32(st, v[0]);
          tmem_ld32(st + 32, v[1]);
          tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int s = min(seg0 + g, segs - 1);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float x = __uint_as_float(v[g >> 1][16 * (g & 1) + j]);
              top = fmaxf(top, key0 + 16 * g + j < lim ? x : -INFINITY);
            }
            m = fmaxf(m, top == -INFINITY ? top : fmaf(top, f * seg_k[s], seg_lv[s]));
          }
        }
        weigh();
        if (__any_sync(0xffffffffu, mx > m + KT_SLACK)) {  // m may be minus infinity
          const float top = fmaxf(m, mx), alpha = m == top ? 1.f : ex2(m - top);
          m = top;
          l *= alpha;
          if (i > 0) {
            mbar_wait(smem_addr(&bars.o_full[half][(i - 1) & 1]), ((i - 1) >> 1) & 1, abort_flag, a.wait_cycles);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t v[16];
              tmem_ld16(ot + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
              tmem_st_words(ot + c, v);
            }
          }
          weigh();
        }
        l += part_l;
        tmem_st32(st, w);  // over the scores just read
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_addr(&bars.p_full[half][i & 1]));
      }
      // join the two halves' sums: each finishes half of the dimensions of every row
      float* other_l = red + 2 * KT_ROWS;
      red[half * KT_ROWS + r] = m;
      other_l[half * KT_ROWS + r] = l;
      if (n > 0) {
        mbar_wait(smem_addr(&bars.o_full[0][(n - 1) & 1]), ((n - 1) >> 1) & 1, abort_flag, a.wait_cycles);
        mbar_wait(smem_addr(&bars.o_full[1][(n - 1) & 1]), ((n - 1) >> 1) & 1, abort_flag, a.wait_cycles);
      }
      tc_fence_after();
      row_barrier();
      const float m0 = red[r], m1 = red[KT_ROWS + r];
      m = fmaxf(m0, m1);
      const float f0 = m0 == m ? 1.f : ex2(m0 - m), f1 = m1 == m ? 1.f : ex2(m1 - m);
      l = other_l[r] * f0 + other_l[KT_ROWS + r] * f1;
      const uint64_t f02 = f2(f0, f0), f12 = f2(f1, f1);
      const uint32_t at = tmem + lanes + O_AT + half * NL;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t v[2][NL];
        if (n > 0) {
          tmem_ld_cols(at + t * (D / 4), v[0]);
          tmem_ld_cols(at + 128 + t * (D / 4), v[1]);
          tmem_ld_wait();
        }
#pragma unroll
        for (int j = 0; j < NL / 2; ++j)
          o[t * NL / 2 + j] = n > 0 ? f2_fma(f2(v[1][2 * j], v[1][2 * j + 1]), f12,
                                             f2_fma(f2(v[0][2 * j], v[0][2 * j + 1]), f02, 0)) : 0;
      }
    }

    if (bars.nans) {  // NaN codes of V entered the products as 0: put back what the row sees
      for (int key = max(c0, kmin & ~(KT_KEYS - 1)); key < min(lim, c1); ++key) {
        const uint8_t* p = a.c.v + seg_at[(key - c0) >> 4] + (key & 15) * D + half * HD;
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) {
          const int d = 4 * (2 * i % NL) + 2 * i / NL;  // of the pair's first value; the second is 4 behind
          float2 x = f2_parts(o[i]);
          if ((p[d] & 0x7f) == 0x7f) x.x = __int_as_float(0x7fffffff);
          if ((p[d + 4] & 0x7f) == 0x7f) x.y = __int_as_float(0x7fffffff);
          o[i] = f2(x.x, x.y);
        }
      }
    }
    if (!whole) l = __int_as_float(0x7fffffff);  // the sequence's length did not fit
    else if (l == 0.f && lim > c0) m = KV_ALL_LOW;
    // through shared memory (the operands are done with), for whole lines on the way out
    float* stage = reinterpret_cast<float*>(smem + C::STAGE_OFF);
    const auto value = [&](int i) { return i & 1 ? f2_parts(o[i >> 1]).y : f2_parts(o[i >> 1]).x; };
#pragma unroll
    for (int j = 0; j < NL; ++j)
      reinterpret_cast<float4*>(stage + r * C::STAGE_LD + half * HD)[j] =
          make_float4(value(j), value(NL + j), value(2 * NL + j), value(3 * NL + j));
    row_barrier();  // red has been read
    if (half == 0) reinterpret_cast<float2*>(red)[r] = make_float2(m - LIFT, l);
  } else if (warp < 8 + C::CODE_WARPS) {
    // ------------------------------------------------------------ codes
    KtCodes<D, C::CODE_WARPS> codes(a.c, seg_at, segs, warp - 8, lane);
    if (n > 0) {
      codes.load_k(0);
      codes.load_v(0);
    }
    for (int i = 0; i < n; ++i) {
      // S and O of tile i - 2 are done with the buffers
      if (i >= 2 && !mbar_wait(smem_addr(&bars.s_full[i & 1]), ((i >> 1) - 1) & 1, abort_flag, a.wait_cycles)) break;
      codes.put_k(smem + C::K_OFF + (i & 1) * C::K_BYTES);
      fence_proxy_async();
      if (!a.withhold || i + 1 < n) mbar_arrive(smem_addr(&bars.k_full[i & 1]));
      if (i + 1 < n) codes.load_k(i + 1);
      if (i >= 2 && !mbar_wait(smem_addr(&bars.o_full[0][i & 1]), ((i >> 1) - 1) & 1, abort_flag, a.wait_cycles)) break;
      if (!PAIR && i >= 2 && !mbar_wait(smem_addr(&bars.o_full[1][i & 1]), ((i >> 1) - 1) & 1, abort_flag, a.wait_cycles)) break;
      // not every row sees every key of the tile: 0 * NaN must not reach the others
      if (c0 + (i + 1) * KT_KEYS > kmin && codes.drop_nans()) bars.nans = 1;
      codes.put_v(smem + C::V_OFF + (i & 1) * C::V_BYTES);
      fence_proxy_async();
      mbar_arrive(smem_addr(&bars.v_full[i & 1]));
      if (i + 1 < n) codes.load_v(i + 1);
    }
  } else {
    // --------------------------------------------------------- products
    const uint32_t leader = elect_leader();
    // The warp's instructions stand between a tile's weights and the next scores: buffers are
    // compile-time numbers and descriptors their low words from a common base, so that a
    // product costs little more than its issue.
    constexpr uint32_t id_s = idesc_f16(KT_ROWS, KT_KEYS), id_o = idesc_f16(KT_ROWS, D);
    constexpr int HALVES = PAIR ? 1 : 2;
    const uint64_t base = sw128_desc(smem_addr(smem));
    const uint32_t lo = (uint32_t)base, hi = (uint32_t)(base >> 32);
    int si = 0, oi[2] = {0, 0};  // products issued
    const auto wait = [&](uint64_t& bar, int i) { return mbar_wait(smem_addr(&bar), (i >> 1) & 1, abort_flag, a.wait_cycles); };
    const auto issue_s = [&](auto buffer) {
      constexpr int B = decltype(buffer)::value;
      tc_fence_after();
#pragma unroll
      for (int pl = 0; pl < (PAIR ? 2 : 1); ++pl)
#pragma unroll
        for (int p = 0; p < C::PANELS; ++p)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_ss_lo(leader, tmem + B * S_COLS, lo + (C::Q_OFF + pl * C::Q_PLANE + p * KT_ROWS * 128) / 16 + 2 * k,
                          lo + (C::K_OFF + B * C::K_BYTES + p * KT_KEYS * 128) / 16 + 2 * k, hi, id_s, pl || p || k);
      if (leader) mma_commit(smem_addr(&bars.s_full[B]));
      ++si;
    };
    // fp32 rows: the whole tile's product, alone in its buffer; bf16 rows: that of one half
    // of the keys, added to the half's sum
    const auto issue_o = [&](auto buffer, auto half, bool add) {
      constexpr int B = decltype(buffer)::value, H = decltype(half)::value;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < (PAIR ? 8 : 4); ++k) {  // 16 keys each
        const int ks = PAIR ? k : 4 * H + k;
        const uint32_t v = lo + (C::V_OFF + B * C::V_BYTES + (ks >> 2) * D * 128) / 16 + 2 * (ks & 3);
        if constexpr (PAIR) {
          const uint32_t p = tmem + B * S_COLS + 16 * k;  // the weights, then their low parts, lie over the scores
          mma_f16_ts_lo(leader, tmem + O_AT + B * 128, p, v, hi, id_o, k > 0);
          mma_f16_ts_lo(leader, tmem + O_AT + B * 128, p + 8, v, hi, id_o, true);
        } else {
          mma_f16_ts_lo(leader, tmem + O_AT + H * 128, tmem + B * S_COLS + 64 * H + 8 * k, v, hi, id_o, k > 0 || add);
        }
      }
      if (leader) mma_commit(smem_addr(&bars.o_full[H][B]));
      ++oi[H];
    };
    const auto tile = [&](int i, auto buffer) {
      constexpr int B = decltype(buffer)::value;
      if (!wait(bars.v_full[B], i) || (PAIR && i >= 2 && !wait(bars.o_free[B], i - 2))) return false;
      if (!wait(bars.p_full[0][B], i)) return false;
      issue_o(buffer, std::integral_constant<int, 0>{}, i > 0);
      if constexpr (!PAIR) {
        if (!wait(bars.p_full[1][B], i)) return false;
        issue_o(buffer, std::integral_constant<int, 1>{}, i > 0);
      }
      if (i + 2 >= n) return true;
      // the next scores of this buffer go over the weights: their products must be done
      if (!wait(bars.k_full[B], i + 2) || !wait(bars.o_full[0][B], i)) return false;
      if (!PAIR && !wait(bars.o_full[1][B], i)) return false;
      issue_s(buffer);
      return true;
    };
    const std::integral_constant<int, 0> even{};
    const std::integral_constant<int, 1> odd{};
    bool ok = n == 0 || mbar_wait(smem_addr(&bars.q_full), 0, abort_flag, a.wait_cycles);
    if (n > 0 && ok && (ok = wait(bars.k_full[0], 0))) issue_s(even);
    if (n > 1 && ok && (ok = wait(bars.k_full[1], 1))) issue_s(odd);
    for (int i = 0; i < n && ok; i += 2) {
      ok = tile(i, even);
      if (ok && i + 1 < n) ok = tile(i + 1, odd);
    }
    if (!ok) {
      for (int i = si > 2 ? si - 2 : 0; i < si; ++i) mbar_drain(smem_addr(&bars.s_full[i & 1]), (i >> 1) & 1);
      for (int h = 0; h < HALVES; ++h)
        for (int i = oi[h] > 2 ? oi[h] - 2 : 0; i < oi[h]; ++i)
          mbar_drain(smem_addr(&bars.o_full[h][i & 1]), (i >> 1) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(a.c.status, RTR_DEV_TIMEOUT);  // whoever's wait ran out
  if (warp == 8 + C::CODE_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // D / 4 threads a row; every warp takes rows in turn
  const float* stage = reinterpret_cast<const float*>(smem + C::STAGE_OFF);
  const float2* ml = reinterpret_cast<const float2*>(red);
  constexpr int LPR = D / 4, RPI = 32 / LPR, WARPS = C::THREADS / 32;
  const int col = lane % LPR;
  const auto finish = [&](int row, float m, float l, float4 x) {
    const int64_t rh = row_out[row];
    l = kv_whole_sum(m, l);
    const bool sees = l != 0.f;
    const float inv = sees ? 1.0f / l : 0.f;
    x = sees ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
    T* p = static_cast<T*>(a.out) + rh * D + 4 * col;
    if constexpr (PAIR) {
      *reinterpret_cast<float4*>(p) = x;
    } else {
      const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(b);
    }
    if (a.lse && col == 0) a.lse[rh] = sees ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  };
  if (!a.cluster) {
    for (int row = warp * RPI + lane / LPR; row < rows; row += WARPS * RPI) {
      const float4 x = *reinterpret_cast<const float4*>(stage + row * C::STAGE_LD + 4 * col);
      const float2 v = ml[row];
      if (a.splits == 1) {
        finish(row, v.x, v.y, x);
      } else {
        const int64_t at = (int64_t)row_out[row] * a.splits + split;
        reinterpret_cast<float4*>(a.part + at * D)[col] = x;
        if (col == 0) a.ml[at] = v;
      }
    }
    return;
  }
  // The cluster's blocks share out the rows: block `row % splits` gets the row from all of
  // them.  Stores into the other blocks' shared memory need no answer; reading it the other way
  // round, 64 KB a block, took 6,100 cycles, this 3,000.
  cluster_sync_all();  // every block is done with its operands
  const int inverse = (65536 + a.splits - 1) / a.splits;  // row / splits = row * inverse >> 16 for these few rows
  const int each = ((KT_ROWS - 1) * inverse >> 16) + 1;
  const uint32_t recv = smem_addr(smem), recv_ml = recv + C::RECV_ROWS * D * 4;
#pragma unroll 4
  for (int row = warp * RPI + lane / LPR; row < rows; row += WARPS * RPI) {
    const int nth = row * inverse >> 16, to = row - nth * a.splits, slot_at = split * each + nth;
    st_cluster_f4(cluster_map(recv + (slot_at * D + 4 * col) * 4, to),
                  *reinterpret_cast<const float4*>(stage + row * C::STAGE_LD + 4 * col));
    if (col == 0) st_cluster_f2(cluster_map(recv_ml + slot_at * 8, to), ml[row]);
  }
  __syncwarp();
  cluster_sync_all();
  const float4* sent = reinterpret_cast<const float4*>(smem);
  const float2* sent_ml = reinterpret_cast<const float2*>(smem + C::RECV_ROWS * D * 4);
  for (int i = warp * RPI + lane / LPR; split + i * a.splits < rows; i += WARPS * RPI) {
    float2 p[KV_CLUSTER];
    float4 v[KV_CLUSTER];
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int s = 0; s < KV_CLUSTER; ++s) {  // without a break: all loads first
      const int from = min(s, a.splits - 1) * each + i;
      p[s] = sent_ml[from];
      v[s] = sent[from * (D / 4) + col];
    }
#pragma unroll
    for (int s = 0; s < KV_CLUSTER; ++s) mt = fmaxf(mt, p[s].x);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < KV_CLUSTER; ++s) {
      if (s >= a.splits) break;
      const float w = p[s].x == mt ? 1.f : ex2(p[s].x - mt);
      lt = fmaf(p[s].y, w, lt);
      x = make_float4(fmaf(v[s].x, w, x.x), fmaf(v[s].y, w, x.y), fmaf(v[s].z, w, x.z), fmaf(v[s].w, w, x.w));
    }
    finish(split + i * a.splits, mt, lt, x);
  }
}

template <typename T, int D> static cudaError_t launch_tile(const KvAttn& a, int64_t items, int device, cudaStream_t st) {
  constexpr int smem = KtCfg<D, std::is_same<T, float>::value>::SMEM;
  static_assert(smem <= 227 * 1024, "a block's shared memory");
  static std::atomic<uint64_t> done;
  const cudaError_t e = kv_allow_smem(kv_attn_tile_kernel<T, D>, smem, done, device);
  if (e != cudaSuccess) return e;
  constexpr int threads = KtCfg<D, std::is_same<T, float>::value>::THREADS;
  return kv_launch(kv_attn_tile_kernel<T, D>, dim3((unsigned)items, a.c.kv_heads, a.splits), threads, smem,
                   a.cluster ? a.splits : 1, st, a);
}

cudaError_t kv_attn_tile(const KvAttn& a, int64_t items, bool f32, int device, cudaStream_t st) {
  if (f32)
    return a.c.head_dim == 128 ? launch_tile<float, 128>(a, items, device, st) : launch_tile<float, 64>(a, items, device, st);
  return a.c.head_dim == 128 ? launch_tile<__nv_bfloat16, 128>(a, items, device, st)
                             : launch_tile<__nv_bfloat16, 64>(a, items, device, st);
}

}  // namespace rtr
