// What the kernels of the 8-bit KV cache share: the cache's and a call's
// pointers, where a call's rows sit in the pages, and e4m3 codes.
//
// A page holds `page` tokens of one sequence for every KV head: codes
// [page][head_dim] per head (one scale per page and head, for K and for V).  A
// sequence's j-th page is table[seq][j].  Sequence b holds lens[b] tokens; the
// call's rows starts[b] .. starts[b + 1] - 1 belong to it (equal shares without
// starts).  Everything read from device memory (starts, lens, page numbers) is
// checked against the buffers before it is used; what fails sets a bit in the
// cache's status word and its work is left out.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "rtr_b200.h"

namespace rtr {

// The least and greatest scale: 2^-48 and 2^48 (bit patterns of the floats).
// Attention keeps one running maximum of score + log2(V scale) and gets the
// softmax sum back by dividing by the scale: with a factor of 2^96 at most
// between two pages, a weight that counts (2^-24 of the sum) stays a normal
// float.
constexpr int KV_EXP = 48;

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int64_t page_stride, head_stride, scale_stride;
  int32_t pages, kv_heads, page_shift, head_dim;
  uint32_t* status;
};

struct KvBatch {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;  // null: every sequence has rows / seqs rows
  int64_t table_stride;
  int32_t table_width, seqs, rows;
};

// The rows of one sequence: first row and count; false (with the status bit) when starts
// does not fit the call (kv_find_seq has looked; this is what the addresses come from).
RTR_DEVICE bool kv_rows(const KvBatch& b, int seq, uint32_t* status, int& first, int& count) {
  if (!b.starts) {
    count = b.rows / b.seqs;
    first = seq * count;
    return true;
  }
  first = b.starts[seq];
  const int end = b.starts[seq + 1];
  count = end - first;
  if (first >= 0 && end >= first && end <= b.rows) return true;
  atomicOr(status, RTR_DEV_BAD_LENGTH);
  return false;
}

// Whether a sequence's length fits its table row and holds `least` tokens.
RTR_DEVICE bool kv_len_fits(const KvCache& c, const KvBatch& b, int len, int least) {
  if (len >= least && len <= (int64_t)b.table_width << c.page_shift) return true;
  atomicOr(c.status, RTR_DEV_BAD_LENGTH);
  return false;
}

// Which sequence a work item belongs to, when sequence b's items are those from
// (starts[b] * num >> shift) + b * extra on: found by all threads of the block, each
// looking at some sequences.  -1 for an item behind the last sequence's.  Where any of
// starts does not fit the call the call is refused: -2 for every item, and the status bit.
// (Some sequences of such a call match no item, others match one another's.)
RTR_DEVICE int kv_find_seq(const KvBatch& b, int64_t item, int num, int shift, int extra, uint32_t* status, int* slot,
                           int64_t& item0) {
  if (threadIdx.x == 0) {
    slot[0] = -1;
    slot[1] = 0;
  }
  __syncthreads();
  for (int s = threadIdx.x; s < b.seqs; s += blockDim.x) {
    const int first = b.starts[s], end = b.starts[s + 1];
    if (first < 0 || end < first || end > b.rows) slot[1] = 1;
    const int64_t lo = ((int64_t)first * num >> shift) + (int64_t)s * extra;
    const int64_t hi = ((int64_t)end * num >> shift) + (int64_t)(s + 1) * extra;
    if (item >= lo && item < hi) slot[0] = s;
  }
  __syncthreads();
  if (slot[1]) {
    if (threadIdx.x == 0) atomicOr(status, RTR_DEV_BAD_LENGTH);
    return -2;
  }
  const int seq = slot[0];
  if (seq >= 0) item0 = ((int64_t)b.starts[seq] * num >> shift) + (int64_t)seq * extra;
  return seq;
}

// The page of a sequence's `nth` page, or -1 (with the status bit) where the
// table names none.
RTR_DEVICE int kv_page(const KvCache& c, const KvBatch& b, int seq, int nth) {
  const int p = b.table[(int64_t)seq * b.table_stride + nth];
  if (p >= 0 && p < c.pages) return p;
  atomicOr(c.status, RTR_DEV_BAD_PAGE);
  return -1;
}

// Two codes (low byte first) as fp16 values: exact, NaN stays NaN.
RTR_DEVICE uint32_t e4m3x2_to_f16x2(uint16_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}
// Two values as codes, to nearest even; the caller keeps magnitudes at most 448.
RTR_DEVICE uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace rtr
