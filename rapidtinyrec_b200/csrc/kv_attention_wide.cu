// Attention over the 8-bit KV cache, bf16 rows of 128, where there are enough of them to give
// every SM 256: two tiles of 128 rows a block share the operands that its code warps make.
//
// The mathematics is that of kv_attention_tile.cu, whose two buffers of S wait for the chain
// weights - O - S of one tile.  Here there are four chains: two row tiles, and two halves of a
// tile's 128 keys each.  A row's thread works on one half while the tensor core forms the
// other's sum and next scores, and the two tiles' threads take turns at the exponential unit;
// codes are converted once for 256 rows.  Tensor memory: S and O of either tile, 128 columns
// each; a half's weights lie over its scores.  Weights are computed in one pass with the
// maximum as it stands; only where a score exceeds it by more than 2^KT_SLACK (weights stay below
// 2^15) are O and the sum rescaled and the pass repeated.
//
// 128 keys take a block some 3,200 cycles (exponentials alone 2,048, products 2,048; one row
// tile by itself 2,600: a thread's chain of loads, exponentials and stores), its start and end
// about seven times that.  8 x 1,024 rows at the end of 6,000 keys, 28 / 4 heads: 640 us,
// 1,007 TFLOP/s of what the mask leaves, tiles of 128 rows 801; 1,024 rows at the end of 30,000 keys
// 455 : 634; at head_dim 64 no difference.
#include <cuda_runtime.h>

#include <climits>
#include <type_traits>

#include "engine.h"
#include "kv_attention_tile.cuh"
#include "kv_host.h"

namespace rtr {

constexpr int KW_SEGS = KW_MAX_CHUNK / 16;
constexpr int KW_JOIN = 8;  // rows of a block that joins, a warp each

struct KwCfg {
  static constexpr int D = 128;
  static constexpr int CODE_WARPS = 4;
  static constexpr int THREADS = KT_ROW_THREADS + 32 * CODE_WARPS + 32;
  static constexpr int PANELS = D / 64;                    // 128-byte panels of a q or k row
  static constexpr int Q_TILE = PANELS * KT_ROWS * 128;
  static constexpr int K_BYTES = PANELS * KT_KEYS * 128;
  static constexpr int V_BYTES = 2 * D * 128;
  static constexpr int Q_OFF = 0, K_OFF = 2 * Q_TILE, V_OFF = K_OFF + 2 * K_BYTES;
  static constexpr int SEG_OFF = V_OFF + 2 * V_BYTES;      // int64 offsets, then 3 floats a segment
  static constexpr int ROW_OFF = SEG_OFF + KW_SEGS * 20;   // per row: row of out, keys it sees
  static constexpr int BACK_OFF = ROW_OFF + KW_ROWS * 8;   // per row: from products to scores
  static constexpr int BAR_OFF = BACK_OFF + KW_ROWS * 4;
  // the finished rows lie over the operands, as bf16 or fp32
  static constexpr int STAGE_LD16 = D * 2 + 16, STAGE_LD32 = D * 4 + 16;
  static_assert(KW_ROWS * STAGE_LD32 <= SEG_OFF, "the finished rows fit over the operands");
  static constexpr int SMEM = BAR_OFF + 256 + 1024;        // 1024: alignment of the operands
};

struct KwBars {
  uint64_t q_full, k_full[2], v_full[2], k_free[2], v_free[2];  // [buffer of the keys]
  uint64_t s_full[2][2], p_full[2][2], o_full[2][2];            // [row tile][half of the keys]: one phase a key tile
  uint32_t tmem;
  int abort_flag;
  int nans;  // V has NaN codes in a tile that not every row sees as a whole
};
static_assert(sizeof(KwBars) <= 256, "barriers fit their part of shared memory");

// Bits of the first `n` of up to 32 keys.
RTR_DEVICE uint32_t seen_keys(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }

__global__ void __launch_bounds__(KwCfg::THREADS, 1) kv_attn_wide_kernel(const KvAttn a, const KwShare w) {
  using C = KwCfg;
  constexpr int D = C::D;
  extern __shared__ uint8_t kw_smem_raw[];
  __shared__ int slot[2];
  uint8_t* smem = kw_smem_raw + ((1024u - (smem_addr(kw_smem_raw) & 1023u)) & 1023u);
  int64_t* seg_at = reinterpret_cast<int64_t*>(smem + C::SEG_OFF);
  float* seg_k = reinterpret_cast<float*>(seg_at + KW_SEGS);
  float* seg_lv = seg_k + KW_SEGS;
  float* seg_iv = seg_lv + KW_SEGS;
  int* row_out = reinterpret_cast<int*>(smem + C::ROW_OFF);
  int* row_lim = row_out + KW_ROWS;
  float* back = reinterpret_cast<float*>(smem + C::BACK_OFF);
  KwBars& bars = *reinterpret_cast<KwBars*>(smem + C::BAR_OFF);
  volatile int* abort_flag = &bars.abort_flag;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  // the first blocks take an item (row tile and KV head) as a whole, the others a stretch of its keys
  const bool alone = (int)blockIdx.x < w.whole;
  const int piece = alone ? 0 : (int)blockIdx.x - w.whole;
  const int tail = piece / a.splits, split = piece - tail * a.splits;
  const int at = alone ? (int)blockIdx.x : w.whole + tail, item = at / a.c.kv_heads, kvh = at - item * a.c.kv_heads;
  pdl_launch_dependents();
  pdl_wait();

  int seq, first = 0, count = 0;
  int64_t item0 = 0;
  if (a.b.starts) {
    seq = kv_find_seq(a.b, item, a.group, 8, 1, a.c.status, slot, item0);
  } else {
    seq = item / a.per_seq;
    item0 = (int64_t)seq * a.per_seq;
  }
  int len = seq < 0 ? 0 : a.b.lens[seq];
  if (seq >= 0 && !kv_rows(a.b, seq, a.c.status, first, count)) count = 0;
  const int nrows = count * a.group;
  const int64_t row0 = (item - item0) * KW_ROWS;
  if (seq < 0 || row0 < 0 || row0 >= nrows) {
    if (!alone && split == 0 && tid < KW_ROWS) w.row[tail * KW_ROWS + tid] = -1;  // nothing to join
    return;
  }
  const int r0 = (int)row0, rows = min(KW_ROWS, nrows - r0);
  const int tiles = rows > KT_ROWS ? 2 : 1;
  constexpr int QLPR = D / 8, QRPI = 32 / QLPR, QLOADS = 32 / QRPI;  // q: lanes of a row, rows of a load
  const int token0 = r0 / a.group, head0 = r0 - token0 * a.group;  // of the block's first row
  // token and head (of the group) of a row of the block
  const auto place = [&](int row, int& token, int& head) {
    const int t = kv_div(a, head0 + min(row, rows - 1));
    token = token0 + t;
    head = head0 + min(row, rows - 1) - t * a.group;
  };
  const bool whole = kv_len_fits(a.c, a.b, len, 0);
  if (!whole) len = 0;  // the sequence's rows become NaN
  const auto limit = [&](int row) { return a.causal && count > 1 ? max(0, len - count + min(row, nrows - 1) / a.group + 1) : len; };
  // keys of a stretch: the item's own, so that a short sequence's stretches are alike too
  const int kmin = limit(r0), kmax = limit(r0 + KW_ROWS - 1);
  const int per = ((kmax + KT_KEYS - 1) / KT_KEYS + a.splits - 1) / a.splits * KT_KEYS;
  const int c0 = (int)min((int64_t)split * per, (int64_t)kmax), c1 = alone ? kmax : c0 + min(kmax - c0, per);
  if (!alone && split == 0 && tid < KW_ROWS) {
    int token, head;
    place(tid, token, head);
    w.row[tail * KW_ROWS + tid] = tid < rows ? (first + token) * a.heads + kvh * a.group + head : -1;
  }
  if (c1 <= c0 && split > 0) {  // a stretch behind the last key (the first one reports rows that see nothing)
    if (tid < rows) a.ml[(int64_t)(tail * KW_ROWS + tid) * a.splits + split] = make_float2(-INFINITY, 0.f);
    return;
  }
  // q comes as it is to its place in the operand, where the thread that fetched it turns it into
  // fp16; a warp takes 32 rows
  const auto q_at = [&](int row, int col) {
    return smem + C::Q_OFF + (row >> 7) * C::Q_TILE + (col >> 3) * KT_ROWS * 128 + sw_at(row & (KT_ROWS - 1), col & 7);
  };
  if (warp < 8) {
#pragma unroll 2
    for (int j = 0; j < QLOADS; ++j) {
      const int row = warp * 32 + j * QRPI + lane / QLPR;
      int token, head;
      place(row, token, head);
      cp_async16(q_at(row, lane % QLPR), static_cast<const __nv_bfloat16*>(a.q) + (int64_t)(first + token) * a.q_token +
                                             (kvh * a.group + head) * D + (lane % QLPR) * 8, row < rows);
    }
    cp_async_commit();
  }
  const int n = c1 > c0 ? (c1 - c0 + KT_KEYS - 1) / KT_KEYS : 0;
  const int segs = c1 > c0 ? (c1 - c0 + 15) / 16 : 0;  // 16-key segments of the stretch

  if (tid == 0) {
    mbar_init(smem_addr(&bars.q_full), KT_ROW_THREADS);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&bars.k_full[i]), 32 * C::CODE_WARPS);
      mbar_init(smem_addr(&bars.v_full[i]), 32 * C::CODE_WARPS);
      mbar_init(smem_addr(&bars.k_free[i]), 1);
      mbar_init(smem_addr(&bars.v_free[i]), 1);
      for (int g = 0; g < 2; ++g) {
        mbar_init(smem_addr(&bars.s_full[g][i]), 1);
        mbar_init(smem_addr(&bars.o_full[g][i]), 1);
        mbar_init(smem_addr(&bars.p_full[g][i]), KT_ROWS);
      }
    }
    bars.nans = 0;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 + C::CODE_WARPS) tmem_alloc(smem_addr(&bars.tmem), 512);
  if (tid < KW_ROWS) {
    int token, head;
    place(tid, token, head);
    row_out[tid] = (first + token) * a.heads + kvh * a.group + head;
    row_lim[tid] = a.causal ? max(0, len - count + token + 1) : len;
  }
  kt_segments(a, seq, kvh, c0, segs, C::THREADS - 1 - tid, C::THREADS, seg_at, seg_k, seg_lv, seg_iv);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(bars.tmem);
  constexpr uint32_t O_AT = 2 * KT_KEYS;

  if (warp < 8) {
    // ------------------------------------------------------------- rows
    const int g = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    cp_async_wait<0>();
    constexpr int STEP = 4;
#pragma unroll 1
    for (int j0 = 0; j0 < QLOADS; j0 += STEP) {  // each row times a power of two; magnitudes order as their bits do
      const int row0 = warp * 32 + j0 * QRPI + lane / QLPR, col = lane % QLPR;
      uint4 u[STEP];
      uint32_t top[STEP];
#pragma unroll
      for (int j = 0; j < STEP; ++j) u[j] = *reinterpret_cast<const uint4*>(q_at(row0 + j * QRPI, col));
#pragma unroll
      for (int j = 0; j < STEP; ++j) {
        const uint32_t mask = 0x7fff7fffu;
        const uint32_t t = __vmaxu2(__vmaxu2(u[j].x & mask, u[j].y & mask), __vmaxu2(u[j].z & mask, u[j].w & mask));
        top[j] = max(t << 16, t & 0xffff0000u);
      }
#pragma unroll
      for (int o = QLPR / 2; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < STEP; ++j) top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
#pragma unroll
      for (int j = 0; j < STEP; ++j) {
        const int row = row0 + j * QRPI, e = kv_row_exponent(__uint_as_float(top[j]));
        const float up = copysignf(kv_pow2(-e), a.factor);  // the factor back stays positive
        if (col == 0) back[row] = kv_pow2(e) * fabsf(a.factor);
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          h[i] = pack_f16(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
        *reinterpret_cast<uint4*>(q_at(row, col)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    fence_proxy_async();
    mbar_arrive(smem_addr(&bars.q_full));
    __syncwarp();
    const float f = back[tid];  // back to the score, in units of log2; positive
    const int lim = row_lim[tid], gmin = limit(r0 + g * KT_ROWS);
    const bool active = g < tiles;
    const uint32_t st = tmem + lanes + g * KT_KEYS, ot = tmem + lanes + O_AT + g * 128;
    float m = -INFINITY, l = 0.f;

    bool ready = false;  // the next half's scores are there: asked early, the answer takes 80 cycles
    for (int i = 0; i < n && active; ++i) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {  // halves of the tile's keys
        if (!ready) mbar_wait(smem_addr(&bars.s_full[g][h]), i & 1, abort_flag, a.wait_cycles);
        tc_fence_after();
        const uint32_t sh = st + 64 * h;
        const int key0 = c0 + i * KT_KEYS + 64 * h, seg0 = i * 8 + 4 * h;
        const bool border = key0 + 64 > gmin;
        uint32_t w[32];
        float mx, part_l;
        // One pass with the maximum as it stands, which also finds the keys' own.
        const auto weigh_keys = [&](float u, auto at_border) {
          constexpr bool BORDER = decltype(at_border)::value;
          uint32_t z[2][16];
          tmem_ld16(sh, z[0]);
          mx = -INFINITY;
          part_l = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int s = min(seg0 + c, segs - 1);
            const float kf = f * seg_k[s], lv = seg_lv[s], iv = seg_iv[s];
            const uint64_t kf2 = f2(kf, kf), lv2 = f2(lv - u, lv - u);
            const uint32_t seen = BORDER ? seen_keys(lim - key0 - 16 * c) : 0xffffffffu;
            tmem_ld_wait();
            uint32_t(&x)[16] = z[c & 1];
            if (c < 3) tmem_ld16(sh + 16 * (c + 1), z[(c + 1) & 1]);
            float top = -INFINITY;
            uint64_t sums = 0;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              float2 t = make_float2(__uint_as_float(x[j]), __uint_as_float(x[j + 1]));
              float2 y = f2_parts(f2_fma(f2(x[j], x[j + 1]), kf2, lv2));
              if constexpr (BORDER) {  // also after the product: the scales of a page that the row does not see may be anything
                if (!(seen >> j & 1)) t.x = y.x = -INFINITY;
                if (!(seen >> (j + 1) & 1)) t.y = y.y = -INFINITY;
              }
              top = fmaxf(top, fmaxf(t.x, t.y));
              y.x = ex2(y.x);
              y.y = ex2(y.y);
              sums = f2_add(sums, f2(y.x, y.y));
              w[8 * c + j / 2] = pack_f16(y.x, y.y);
            }
            part_l = fmaf(f2_parts(sums).x + f2_parts(sums).y, iv, part_l);
            // the factors are positive: the largest product of a segment gives its largest score
            mx = fmaxf(mx, top == -INFINITY ? top : fmaf(top, kf, lv));
          }
        };
        const auto weigh = [&] {
          const float u = (m == -INFINITY ? 0.f : m) - KT_LIFT;
          if (border) weigh_keys(u, std::true_type{});
          else weigh_keys(u, std::false_type{});
        };
        if (i + h == 0) {
          // nothing to go by: the maximum alone first
          uint32_t z[2][32];
          tmem_ld32(sh, z[0]);
          tmem_ld32(sh + 32, z[1]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int s = min(seg0 + c, segs - 1);
            const uint32_t seen = seen_keys(lim - key0 - 16 * c);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              top = fmaxf(top, seen >> j & 1 ? __uint_as_float(z[c >> 1][16 * (c & 1) + j]) : -INFINITY);
            m = fmaxf(m, top == -INFINITY ? top : fmaf(top, f * seg_k[s], seg_lv[s]));
          }
        }
        weigh();
        if (__any_sync(0xffffffffu, mx > m + KT_SLACK)) {  // m may be minus infinity
          const float top = fmaxf(m, mx), alpha = m == top ? 1.f : ex2(m - top);
          m = top;
          l *= alpha;
          if (i + h > 0) {  // the other half's product is the last that O got
            mbar_wait(smem_addr(&bars.o_full[g][h ^ 1]), (i - 1 + h) & 1, abort_flag, a.wait_cycles);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t x[16];
              tmem_ld16(ot + c, x);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
              tmem_st_words(ot + c, x);
            }
          }
          weigh();
        }
        l += part_l;
        ready = mbar_test(smem_addr(&bars.s_full[g][h ^ 1]), (i + h) & 1);
        tmem_st32(sh, w);  // over the scores just read
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_addr(&bars.p_full[g][h]));
      }
    }
    if (n > 0 && active) mbar_wait(smem_addr(&bars.o_full[g][1]), (n - 1) & 1, abort_flag, a.wait_cycles);
    tc_fence_after();
    row_barrier();  // both tiles are done with the operands
    if (!whole) l = __int_as_float(0x7fffffff);  // the sequence's length did not fit
    else if (l == 0.f && lim > c0) m = KV_ALL_LOW;
    const float lt = alone ? kv_whole_sum(m, l) : l;
    // A whole item: finished values as bf16; a stretch: sums as they are.
    const bool sees = lt != 0.f;
    const float inv = !alone ? 1.f : sees ? 1.0f / lt : 0.f;
    uint8_t* stage = smem + tid * (alone ? C::STAGE_LD16 : C::STAGE_LD32);
    const int64_t rh = row_out[tid];
    if (tid < rows) {
      if (!alone) a.ml[(int64_t)(tail * KW_ROWS + tid) * a.splits + split] = make_float2(m - KT_LIFT, lt);
      else if (a.lse) a.lse[rh] = sees ? (m - KT_LIFT + log2f(lt)) * 0.6931471805599453f : -INFINITY;
    }
    if (active) {
      const int nan0 = bars.nans ? max(c0, kmin & ~(KT_KEYS - 1)) : INT_MAX;
#pragma unroll 1
      for (int j = 0; j < D / 32; ++j) {  // dimensions 32 j ..: 4 d + t is column t (D / 4) + d
        uint32_t v[4][8];
        if (n > 0) {
#pragma unroll
          for (int t = 0; t < 4; ++t) tmem_ld_cols(ot + t * (D / 4) + 8 * j, v[t]);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < 8; ++d) v[t][d] = 0;
        }
        uint32_t bad = 0;  // NaN codes of V entered the products as 0: put back what the row sees
        for (int key = nan0; key < min(lim, c1); ++key) {
          const uint8_t* p = a.c.v + seg_at[(key - c0) >> 4] + (key & 15) * D + 32 * j;
#pragma unroll 1
          for (int d = 0; d < 32; ++d) bad |= (uint32_t)((p[d] & 0x7f) == 0x7f) << d;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          float x[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            x[t] = bad >> (4 * d + t) & 1 ? __int_as_float(0x7fffffff) : __uint_as_float(v[t][d]);
            x[t] = alone && !sees ? 0.f : x[t] * inv;
          }
          if (alone) {
            const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
            *reinterpret_cast<uint2*>(stage + 64 * j + 8 * d) = *reinterpret_cast<const uint2*>(b);
          } else {
            *reinterpret_cast<float4*>(stage + 128 * j + 16 * d) = make_float4(x[0], x[1], x[2], x[3]);
          }
        }
      }
    }
  } else if (warp < 8 + C::CODE_WARPS) {
    // ------------------------------------------------------------ codes
    KtCodes<D, C::CODE_WARPS> codes(a.c, seg_at, segs, warp - 8, lane);
    if (n > 0) {
      codes.load_k(0);
      codes.load_v(0);
    }
    for (int i = 0; i < n; ++i) {
      // the products of tile i - 2 are done with the buffers
      if (i >= 2 && !mbar_wait(smem_addr(&bars.k_free[i & 1]), ((i >> 1) - 1) & 1, abort_flag, a.wait_cycles)) break;
      codes.put_k(smem + C::K_OFF + (i & 1) * C::K_BYTES);
      fence_proxy_async();
      if (!a.withhold || i + 1 < n) mbar_arrive(smem_addr(&bars.k_full[i & 1]));
      if (i + 1 < n) codes.load_k(i + 1);
      if (i >= 2 && !mbar_wait(smem_addr(&bars.v_free[i & 1]), ((i >> 1) - 1) & 1, abort_flag, a.wait_cycles)) break;
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
    // Four chains, one for each row tile and half of the keys: a chain's next scores go over its
    // weights once their product is done, while its rows' threads work on the other half.
    // Buffers are compile-time numbers and descriptors their low words from a common base.
    constexpr uint32_t id_s = idesc_f16(KT_ROWS, 64), id_o = idesc_f16(KT_ROWS, D);
    const uint64_t base = sw128_desc(smem_addr(smem));
    const uint32_t lo = (uint32_t)base, hi = (uint32_t)(base >> 32);
    int si[4] = {0, 0, 0, 0}, oi[4] = {0, 0, 0, 0};  // products issued, by chain
    const auto wait = [&](uint64_t& bar, int phase) { return mbar_wait(smem_addr(&bar), phase & 1, abort_flag, a.wait_cycles); };
    const auto issue_s = [&](auto buffer, auto chain) {
      constexpr int B = decltype(buffer)::value, G = decltype(chain)::value & 1, H = decltype(chain)::value >> 1;
      tc_fence_after();
#pragma unroll
      for (int p = 0; p < C::PANELS; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_ss_lo(leader, tmem + G * KT_KEYS + 64 * H, lo + (C::Q_OFF + G * C::Q_TILE + p * KT_ROWS * 128) / 16 + 2 * k,
                        lo + (C::K_OFF + B * C::K_BYTES + p * KT_KEYS * 128 + 64 * H * 128) / 16 + 2 * k, hi, id_s, p || k);
      if (leader) mma_commit(smem_addr(&bars.s_full[G][H]));
      ++si[decltype(chain)::value];
    };
    const auto issue_o = [&](auto buffer, auto chain, bool add) {
      constexpr int B = decltype(buffer)::value, G = decltype(chain)::value & 1, H = decltype(chain)::value >> 1;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 4; ++k)  // 16 keys each
        mma_f16_ts_lo(leader, tmem + O_AT + G * 128, tmem + G * KT_KEYS + 64 * H + 8 * k,
                      lo + (C::V_OFF + B * C::V_BYTES + H * D * 128) / 16 + 2 * k, hi, id_o, H > 0 || k > 0 || add);
      if (leader) mma_commit(smem_addr(&bars.o_full[G][H]));
      ++oi[decltype(chain)::value];
    };
    const std::integral_constant<int, 0> c0_{};
    const std::integral_constant<int, 1> c1_{};
    const std::integral_constant<int, 2> c2_{};
    const std::integral_constant<int, 3> c3_{};
    // the product of a chain's weights of tile i, then its scores of the next one
    const auto step = [&](int i, auto buffer, auto next, auto chain) {
      constexpr int B = decltype(buffer)::value, G = decltype(chain)::value & 1, H = decltype(chain)::value >> 1;
      if (G >= tiles) return true;
      if (!wait(bars.p_full[G][H], i)) return false;
      issue_o(buffer, chain, i > 0);
      if (i + 1 >= n) return true;
      if (!wait(bars.k_full[B ^ 1], (i + 1) >> 1) || !wait(bars.o_full[G][H], i)) return false;
      issue_s(next, chain);
      return true;
    };
    const auto keys = [&](int i, auto buffer, auto next) {
      constexpr int B = decltype(buffer)::value;
      if (!wait(bars.v_full[B], i >> 1)) return false;
      if (!step(i, buffer, next, c0_) || !step(i, buffer, next, c1_)) return false;
      if (!step(i, buffer, next, c2_) || !step(i, buffer, next, c3_)) return false;
      // tile i's V, the next tile's K; nothing arrives for which no one waits
      if (leader && i + 2 < n) mma_commit(smem_addr(&bars.v_free[B]));
      if (leader && i + 3 < n) mma_commit(smem_addr(&bars.k_free[B ^ 1]));
      return true;
    };
    bool ok = n == 0 || (wait(bars.q_full, 0) && wait(bars.k_full[0], 0));
    if (n > 0 && ok) {
      issue_s(c0_, c0_);
      if (tiles > 1) issue_s(c0_, c1_);
      issue_s(c0_, c2_);
      if (tiles > 1) issue_s(c0_, c3_);
      if (leader && n > 2) mma_commit(smem_addr(&bars.k_free[0]));
    }
    for (int i = 0; i < n && ok; i += 2) {
      ok = keys(i, c0_, c1_);
      if (ok && i + 1 < n) ok = keys(i + 1, c1_, c0_);
    }
    if (!ok) {
      for (int c = 0; c < 4; ++c) {
        if (si[c]) mbar_drain(smem_addr(&bars.s_full[c & 1][c >> 1]), (si[c] - 1) & 1);
        if (oi[c]) mbar_drain(smem_addr(&bars.o_full[c & 1][c >> 1]), (oi[c] - 1) & 1);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(a.c.status, RTR_DEV_TIMEOUT);  // whoever's wait ran out
  if (warp == 8 + C::CODE_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // whole lines on the way out
  const int units = alone ? D / 8 : D / 4, ld = alone ? C::STAGE_LD16 : C::STAGE_LD32;  // 16 bytes of a row
#pragma unroll 4
  for (int i = tid; i < rows * units; i += C::THREADS) {
    const int row = i / units, unit = i % units;
    uint8_t* to = alone ? static_cast<uint8_t*>(a.out) + (int64_t)row_out[row] * D * 2
                        : reinterpret_cast<uint8_t*>(a.part + ((int64_t)(tail * KW_ROWS + row) * a.splits + split) * D);
    *reinterpret_cast<uint4*>(to + 16 * unit) = *reinterpret_cast<const uint4*>(smem + row * ld + 16 * unit);
  }
}

// Joins the stretches of the items that were split: a warp has a row.
__global__ void __launch_bounds__(32 * KW_JOIN) kv_attn_wide_join_kernel(const KvAttn a, const KwShare w) {
  constexpr int D = KwCfg::D;
  static_assert(D == 4 * 32, "a lane has four columns");
  pdl_launch_dependents();
  pdl_wait();
  const int col = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * KW_JOIN + (threadIdx.x >> 5);
  const int rh = w.row[row];
  if (rh < 0) return;
  const float2* ml = a.ml + row * a.splits;
  const float4* part = reinterpret_cast<const float4*>(a.part + row * a.splits * D) + col;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[s].x);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float2 p = ml[s];
    if (p.y == 0.f) continue;  // nothing seen there means nothing written to part
    const float f = p.x == m ? 1.f : ex2(p.x - m);
    const float4 v = part[s * 32];
    l = fmaf(p.y, f, l);
    x = make_float4(fmaf(v.x, f, x.x), fmaf(v.y, f, x.y), fmaf(v.z, f, x.z), fmaf(v.w, f, x.w));
  }
  l = kv_whole_sum(m, l);
  const bool sees = l != 0.f;
  const float inv = sees ? 1.0f / l : 0.f;
  x = sees ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
  const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
  reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (int64_t)rh * D)[col] = *reinterpret_cast<const uint2*>(b);
  if (a.lse && col == 0) a.lse[rh] = sees ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

cudaError_t kv_attn_wide(const KvAttn& a, const KwShare& w, int device, cudaStream_t st) {
  static_assert(KwCfg::SMEM <= 227 * 1024, "a block's shared memory");
  static std::atomic<uint64_t> done;
  cudaError_t e = kv_allow_smem(kv_attn_wide_kernel, KwCfg::SMEM, done, device);
  if (e != cudaSuccess) return e;
  e = kv_launch(kv_attn_wide_kernel, dim3(w.whole + w.tails * a.splits), KwCfg::THREADS, KwCfg::SMEM, 1, st, a, w);
  if (e != cudaSuccess || !w.tails) return e;
  return kv_launch(kv_attn_wide_join_kernel, dim3(w.tails * (KW_ROWS / KW_JOIN)), 32 * KW_JOIN, 0, 1, st, a, w);
}

}  // namespace rtr
