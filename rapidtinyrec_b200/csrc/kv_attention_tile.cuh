// What the kernels with tiles of query rows on the 5th-generation tensor cores share
// (kv_attention_tile.cu: 128 rows a block, kv_attention_wide.cu: 256): products with their
// operands in shared and tensor memory, pages and scales of a stretch, and the warps that
// turn codes into swizzled fp16 operands.
#pragma once

#include "kv_attention.cuh"

namespace rtr {

constexpr int KT_ROW_THREADS = 256;
constexpr int KT_SEGS = KT_MAX_CHUNK / 16;
// bf16 rows: log2 by which a maximum may be exceeded before the sums are rescaled, and the
// lift that leaves room for it: weights down to 2^-24 of the maximum keep 11 bits, smaller ones
// are off by 2^-35 of it at most.  1,803 rows over 5,603 and 7,025 keys, 28 / 4 heads: 178 us,
// with a slack of 8 and a lift of 7 175, with 4 and 11 180.
constexpr float KT_SLACK = 5.0f, KT_LIFT = 10.0f;

// The products' warp runs as a whole, and one of its threads (the leader) issues: where the
// compiler sees that a warp does not diverge, descriptors and addresses stay in uniform
// registers, which the instructions take; one thread in a branch of its own moved each of
// them there first (a product of 16 keys took 70 cycles to issue, now 20 - 30).
RTR_DEVICE int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// Whether a barrier's phase is complete, without waiting.
RTR_DEVICE bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
RTR_DEVICE uint32_t elect_leader() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// D[tmem] (+)= A . B[smem]^T, kind::f16 (both fp16), A in shared or tensor memory;
// descriptors as low words and their common high word.
RTR_DEVICE void mma_f16_ss_lo(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
RTR_DEVICE void mma_f16_ts_lo(uint32_t leader, uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
RTR_DEVICE void tmem_st_words(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
RTR_DEVICE void tmem_st_words(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
RTR_DEVICE void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }
RTR_DEVICE void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// The row threads of a block.
RTR_DEVICE void row_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// The two warps that have the halves of the same rows.
RTR_DEVICE void halves_barrier(int warp) { asm volatile("bar.sync %0, 64;" ::"r"(2 + warp) : "memory"); }
// Byte of a 16-byte unit of a 128-byte row in a 128B-swizzled operand.
RTR_DEVICE uint32_t sw_at(int row, int unit) { return row * 128 + ((unit ^ (row & 7)) << 4); }

// Pages and scales of a stretch's 16-key segments (a page is a multiple of 16), by threads
// `from`, `from` + `step`, ...
RTR_DEVICE void kt_segments(const KvAttn& a, int seq, int kvh, int c0, int segs, int from, int step, int64_t* seg_at,
                            float* seg_k, float* seg_lv, float* seg_iv) {
  for (int s = from; s < segs; s += step) {
    const int key = c0 + 16 * s;
    const int page = kv_page(a.c, a.b, seq, key >> a.c.page_shift);
    int64_t at = kvh * a.c.head_stride;
    float ks, lv, iv = 0.f;
    ks = lv = __int_as_float(0x7fffffff);  // a page that is not there makes the rows NaN, whatever codes are read
    if (page >= 0) {
      at += page * a.c.page_stride + (int64_t)(key & ((1 << a.c.page_shift) - 1)) * a.c.head_dim;
      ks = kv_k_scale(a.c.k_scale[page * a.c.scale_stride + kvh]);
      kv_v_scale(a.c.v_scale[page * a.c.scale_stride + kvh], lv, iv);
    }
    seg_at[s] = at;
    seg_k[s] = ks;
    seg_lv[s] = lv;
    seg_iv[s] = iv;
  }
}

// One warp's part (of WARPS) in turning a tile's codes into operands: K as [panel of 64
// dims][key][64 dims], V transposed as [64 keys][dim][64 keys], where dimension 4 l + t is
// row t (D / 4) + l.  Loads need no conditions: a segment lies in one page as a whole, and
// what is read of keys behind the last (or of the last segment again) is masked, NaN codes of
// V are taken out by drop_nans.  Ordinary loads: the launch begins before its predecessor,
// which may write these pages, has ended, and what the read-only path serves must not change
// while a kernel runs.
template <int D, int WARPS> struct KtCodes {
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int KP = KT_KEYS * D / 16 / THREADS;       // 16-byte pieces of K a thread: 8 or 4
  static constexpr int LPK = D / 16;                          // threads of a key
  static constexpr int VO = KT_KEYS / 8 * (D / 4) / THREADS;  // (8 keys x 4 dims) blocks of V a thread: 4 or 2
  const uint8_t *k, *v;
  const int64_t* seg_at;
  int segs, cw, lane, piece, key_of, dl;
  uint4 kr[KP];
  uint32_t vr[VO][8];

  // Of K, eight consecutive lanes take four pieces of one panel of two neighbouring keys:
  // their stores then hit all banks.
  RTR_DEVICE KtCodes(const KvCache& c, const int64_t* at, int segments, int warp, int l)
      : k(c.k), v(c.v), seg_at(at), segs(segments), cw(warp), lane(l),
        piece(D == 128 ? (l & 3) + 4 * (l >> 3 & 1) : l & 3),
        key_of(warp * (32 / LPK) + (D == 128 ? 2 * (l >> 4) + (l >> 2 & 1) : l >> 2)), dl(l % (D / 4)) {}
  RTR_DEVICE int octet(int o) const { return (o * WARPS + cw) * (32 / (D / 4)) + lane / (D / 4); }
  RTR_DEVICE void load_k(int i) {
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int rel = i * KT_KEYS + p * (THREADS / LPK) + key_of;
      kr[p] = *reinterpret_cast<const uint4*>(k + seg_at[min(rel >> 4, segs - 1)] + (rel & 15) * D + 16 * piece);
    }
  }
  RTR_DEVICE void load_v(int i) {
#pragma unroll
    for (int o = 0; o < VO; ++o) {
      const int rel = i * KT_KEYS + 8 * octet(o);
      const uint8_t* p = v + seg_at[min(rel >> 4, segs - 1)] + (rel & 8) * D + 4 * dl;
#pragma unroll
      for (int j = 0; j < 8; ++j) vr[o][j] = *reinterpret_cast<const uint32_t*>(p + j * D);
    }
  }
  RTR_DEVICE void put_k(uint8_t* kd) const {
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int key = p * (THREADS / LPK) + key_of;
      const uint32_t w[4] = {kr[p].x, kr[p].y, kr[p].z, kr[p].w};
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[2 * j] = e4m3x2_to_f16x2((uint16_t)w[j]);
        h[2 * j + 1] = e4m3x2_to_f16x2((uint16_t)(w[j] >> 16));
      }
      uint8_t* row = kd + (piece >> 2) * KT_KEYS * 128;
      const int un = 2 * (piece & 3);
      *reinterpret_cast<uint4*>(row + sw_at(key, un)) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(row + sw_at(key, un + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
    }
  }
  // NaN codes of the V on hand become 0; whether there were any.
  RTR_DEVICE bool drop_nans() {
    uint32_t bad = 0;
#pragma unroll
    for (int o = 0; o < VO; ++o)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t nb = nan_bytes(vr[o][j]);
        bad |= nb;
        vr[o][j] &= ~((nb >> 7) * 0xffu);
      }
    return bad != 0;
  }
  RTR_DEVICE void put_v(uint8_t* vd) const {
#pragma unroll
    for (int o = 0; o < VO; ++o) {
      const int oc = octet(o);
      uint32_t h[4][4];  // [dim t][keys 2 j, 2 j + 1]
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = __byte_perm(vr[o][2 * j], vr[o][2 * j + 1], 0x5140);
        const uint32_t y = __byte_perm(vr[o][2 * j], vr[o][2 * j + 1], 0x7362);
        h[0][j] = e4m3x2_to_f16x2((uint16_t)x);
        h[1][j] = e4m3x2_to_f16x2((uint16_t)(x >> 16));
        h[2][j] = e4m3x2_to_f16x2((uint16_t)y);
        h[3][j] = e4m3x2_to_f16x2((uint16_t)(y >> 16));
      }
      // consecutive lanes, consecutive rows
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *reinterpret_cast<uint4*>(vd + (oc >> 3) * D * 128 + sw_at(t * (D / 4) + dl, oc & 7)) =
            make_uint4(h[t][0], h[t][1], h[t][2], h[t][3]);
    }
  }
};

}  // namespace rtr
