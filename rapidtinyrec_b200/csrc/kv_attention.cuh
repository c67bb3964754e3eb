// What the attention kernels over the 8-bit KV cache share (kv_attention.cu: few rows,
// kv_attention_tile.cu: tiles of 128 rows, kv_attention_wide.cu: two such tiles a block).
#pragma once

#include "kv_cache.cuh"
#include "tcgen05.cuh"

namespace rtr {

constexpr int KV_CLUSTER = 8;  // stretches that one cluster joins

struct KvAttn {
  KvCache c;
  KvBatch b;
  const void* q;
  int64_t q_token;     // elements between a token's rows; heads are contiguous
  int heads, group;    // query heads, and those of one KV head
  uint32_t group_inverse;  // ceil(2^32 / group): see kv_div
  int causal;
  float factor;        // softmax scale * log2(e)
  void* out;           // [rows][heads][head_dim]
  float* lse;          // [rows][heads] or null
  float* part;         // [rows * heads][splits][head_dim] when splits > 1
  int* refused;        // with starts, and stretches that a kernel joins: whether the call is refused
  float2* ml;          // [rows * heads][splits]: log2 of the unit of part and of the sum, sum
  int per_seq;         // row tiles of a sequence without starts
  int chunk, splits;   // keys of a block, and the blocks of a row tile
  int cluster;         // the blocks of a row tile are one cluster and join among themselves
  int withhold;        // a test's: the tile kernels do not hand over the last K of a block's keys
  long long wait_cycles;  // the limit of the tile kernels' waits
};

// Weights enter the fp16 operands relative to 2^(maximum - lift): the lift brings the largest
// near fp16's largest, 2^16, since what lies below fp16's smallest normal value, 2^-14, is
// rounded to multiples of 2^-24 and a few keys that outweigh thousands of others (whose values
// may be 0) must not cost those their precision.  Where the maximum is always the running one,
// the lift is 15: weights down to 2^-29 of the largest keep the operand's 11 bits.
constexpr float KA_LIFT = 15.0f;
// The low parts of pairs enter times 2^11, as large as the high ones, where their product has
// an accumulator of its own: 22 bits down to the same 2^-29.
constexpr float KA_LOW = 2048.0f;

// A row's sum l, in units of 2^m.  A row that sees nothing has m = -infinity and l = 0; one that
// sees keys whose scores are all minus infinity (products beyond float's range) has KV_ALL_LOW and
// l = 0: nothing beside a stretch that has more, NaN (0 / 0) where all stretches are so.
constexpr float KV_ALL_LOW = -3.402823466e+38f;
RTR_DEVICE float kv_whole_sum(float m, float l) { return l == 0.f && m != -INFINITY ? __int_as_float(0x7fffffff) : l; }

// v / group for v < 2^32 / group (v is a row's place within some tiles): one multiplication.
// A group of one has no 32-bit inverse.
RTR_DEVICE int kv_div(const KvAttn& a, int v) { return a.group == 1 ? v : (int)__umulhi((uint32_t)v, a.group_inverse); }

// The sums of a cluster's blocks for one row: their joined maximum and sum, and four
// columns.  ml_at: this block's (maximum, sum), x_at: its columns; all loads are issued before
// any is used (one after the other they cost 250 cycles each).
RTR_DEVICE float4 kv_join_cluster(uint32_t ml_at, uint32_t x_at, int splits, float& m, float& l);

RTR_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
RTR_DEVICE float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
RTR_DEVICE float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
RTR_DEVICE float4 kv_join_cluster(uint32_t ml_at, uint32_t x_at, int splits, float& m, float& l) {
  float2 ml[KV_CLUSTER];
  float4 v[KV_CLUSTER];
#pragma unroll
  for (int s = 0; s < KV_CLUSTER; ++s) {
    if (s >= splits) break;
    ml[s] = ld_cluster_f2(cluster_map(ml_at, s));
    v[s] = ld_cluster_f4(cluster_map(x_at, s));
  }
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int s = 0; s < KV_CLUSTER; ++s)
    if (s < splits) m = fmaxf(m, ml[s].x);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int s = 0; s < KV_CLUSTER; ++s) {
    if (s >= splits) break;
    const float w = ml[s].x == m ? 1.f : ex2(ml[s].x - m);
    l = fmaf(ml[s].y, w, l);
    x = make_float4(fmaf(v[s].x, w, x.x), fmaf(v[s].y, w, x.y), fmaf(v[s].z, w, x.z), fmaf(v[s].w, w, x.w));
  }
  return x;
}
RTR_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What is left of two values beside their fp16 parts: exact, in one instruction each.
RTR_DEVICE float2 rest_f16(uint32_t parts, float lo, float hi) {
  float2 r;
  asm("{\n\t.reg .f16 a, b, minus;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 minus, 0xBC00;\n\t"
      "fma.rn.f32.f16 %0, a, minus, %3;\n\tfma.rn.f32.f16 %1, b, minus, %4;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(parts), "f"(lo), "f"(hi));
  return r;
}
// Two fp32 lanes of one instruction.
RTR_DEVICE uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
RTR_DEVICE uint64_t f2(uint32_t lo, uint32_t hi) { return f2(__uint_as_float(lo), __uint_as_float(hi)); }
RTR_DEVICE float2 f2_parts(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
RTR_DEVICE uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
RTR_DEVICE uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RTR_DEVICE uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Whether one of four codes is NaN (0x7f or 0xff).
RTR_DEVICE uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A K scale: negative ones (and NaN) make what uses them NaN.
RTR_DEVICE float kv_k_scale(float ks) { return ks >= 0.f ? ks : __int_as_float(0x7fffffff); }
// A V scale's two uses: log2 of it (an exponent's part) and its reciprocal.  NaN where
// it lies outside [2^-48, 2^48].
RTR_DEVICE void kv_v_scale(float vs, float& log2_scale, float& inverse) {
  const bool fits = vs >= 1.0f / 281474976710656.0f && vs <= 281474976710656.0f;
  log2_scale = fits ? log2f(vs) : __int_as_float(0x7fffffff);
  inverse = fits ? 1.0f / vs : 0.f;
}
// The power of two that brings a row's largest magnitude into [2^13, 2^14), as its
// exponent with the sign turned: the row is multiplied by 2^-e, its scores by 2^e.
RTR_DEVICE int kv_row_exponent(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) - 127 - 13;
  return top > 0.f && top < INFINITY ? max(-100, e) : 0;
}
RTR_DEVICE float kv_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Tiles of 128 rows on the 5th-generation tensor cores (kv_attention_tile.cu).
constexpr int KT_ROWS = 128, KT_KEYS = 128;
constexpr int KT_MAX_CHUNK = 8192;  // keys of a block
cudaError_t kv_attn_tile(const KvAttn& a, int64_t items, bool f32, int device, cudaStream_t st);

// Two such tiles a block, bf16 rows (kv_attention_wide.cu).  Of the items (256 rows and a KV
// head) the first `whole` have a block each, the `tails` others a.splits blocks, each a
// stretch of a.chunk keys: a.part and a.ml are [tails][256][splits].
constexpr int KW_ROWS = 2 * KT_ROWS;
constexpr int KW_MAX_CHUNK = 16384;  // keys of a block
struct KwShare {
  int whole, tails;
  int* row;  // [tails][256]: the (row, head) of out, -1 for none
};
cudaError_t kv_attn_wide(const KvAttn& a, const KwShare& w, int device, cudaStream_t st);

}  // namespace rtr
