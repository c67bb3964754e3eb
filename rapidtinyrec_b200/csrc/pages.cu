// Page numbers handed out and taken back on the GPU: page tables, row offsets, positions and
// slots from the lengths of a batch of sequences.
//
// Mathematics.  n tokens need ceil(n / page) pages.  With need[b] = pages(held + fresh) - pages(held)
// the call's page items are numbered by the running sum of need, its rows by the running
// sum of fresh; item j takes the j-th number from the top of the stack of free pages.  Everything else is a search of an item
// or a row in those two sums.
//
// What bounds it.  Some kilobytes for a step's tokens: the launch and three dependent loads (lengths,
// table or stack, store), with the block's scan between them: 64 sequences, a token each, 2.9 us on the device, of which the
// scan is 1.1; 1,900 sequences 6.1, the scan 2.5.  For prompts the 12 bytes a row are written at L2's rate (127,000 rows: 3.8 us).  So one
// launch does it all: every block sums the lengths itself (they are in L2, and the scan costs less than a second
// launch or a barrier over the grid) and then takes its share of rows and items.  A call that does not fit must
// change nothing, and every block finds that out for itself from the same numbers.
// Taking changes the stack's height alone, which the last block to finish does, by a ticket; a page
// item of the call is read from the stack by whoever needs it, so no block waits for another.
//
// Giving back is all or nothing over values that lie in the table (a page number that is out of
// range, or that no sequence holds), so its blocks have to agree before any of them writes: they are
// one cluster, which marks every page first, then pushes them or takes the marks back (64 sequences 5.2 us: the cluster's
// start and its two barriers are half of it).
#include <cuda_runtime.h>

#include <cooperative_groups.h>

#include "engine.h"
#include "kv_host.h"

namespace rtr {

constexpr int PG_FEW = 256, PG_MANY = 1024;  // threads of a block, up to so many sequences and beyond
constexpr int PG_MAX_SEQS = 16384, PG_BACK_CLUSTER = 8;
constexpr int PG_PER = 2;                    // entries of a table a thread, by which pages given back get blocks
constexpr int PG_HELD = 8;                   // pages given back that a thread remembers

struct PagePool {
  int32_t* free;
  int32_t* count;
  int32_t* marks;
  uint32_t* status;
  uint32_t* ticket;
  int32_t pages, shift;
};

struct PageSeqs {
  int32_t* table;
  int64_t stride;
  int32_t width, seqs;
  const int32_t* held;
};

RTR_DEVICE int pages_of(int tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }  // lengths leave room for a page

// The running sums of two numbers a sequence, by all threads of the block: a[0 .. seqs], b[0 .. seqs]
// (b null: one number).  value(s, x, y) gives sequence s's two numbers and false where it does not fit; the
// result is false where any sequence does not fit or a sum is above its limit (what a and b hold then means nothing).
// A round takes as many sequences as the block has threads.
template <typename F>
RTR_DEVICE bool page_sums(int seqs, int32_t* a, int32_t* b, int64_t limit_a, int64_t limit_b, F&& value) {
  __shared__ longlong2 red[PG_MANY / 32 + 1];  // warps' sums, then what lies before each warp; behind them all that was seen
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  int fits = 1, p = 0, q = 0;
  const auto load = [&](int s) {
    p = q = 0;
    if (s < seqs && !value(s, p, q)) fits = p = q = 0;
  };
  load(tid);
  for (int s0 = 0; s0 < seqs; s0 += blockDim.x) {
    const int s = s0 + tid;
    // a warp's sums in 64 bits, by halves of the numbers; the running ones in 32, which are right where the call fits
    const auto whole = [](int n) {
      return ((int64_t)__reduce_add_sync(0xffffffffu, (unsigned)n >> 16) << 16) + __reduce_add_sync(0xffffffffu, (unsigned)n & 0xffffu);
    };
    const int64_t all_x = whole(p), all_y = b ? whole(q) : 0;
    uint32_t x = p, y = q;
    load(s + blockDim.x);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, x, d), v = b ? __shfl_up_sync(0xffffffffu, y, d) : 0u;
      if (lane >= d) {
        x += u;
        y += v;
      }
    }
    if (lane == 31) red[warp] = make_longlong2(all_x, all_y);
    __syncthreads();
    if (warp == 0) {
      longlong2 m = lane < warps ? red[lane] : make_longlong2(0, 0), sum = m;
      const longlong2 seen = s0 ? red[PG_MANY / 32] : make_longlong2(0, 0);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, sum.x, d), v = __shfl_up_sync(0xffffffffu, sum.y, d);
        if (lane >= d) {
          sum.x += u;
          sum.y += v;
        }
      }
      __syncwarp();
      if (lane < warps) red[lane] = make_longlong2(seen.x + sum.x - m.x, seen.y + sum.y - m.y);
      if (lane == 31) red[PG_MANY / 32] = make_longlong2(seen.x + sum.x, seen.y + sum.y);
    }
    __syncthreads();
    if (s < seqs) {
      a[s + 1] = (int32_t)(x + (uint32_t)red[warp].x);
      if (b) b[s + 1] = (int32_t)(y + (uint32_t)red[warp].y);
    }
    __syncwarp();  // the next round writes the warp's place
  }
  if (tid == 0) {
    a[0] = 0;
    if (b) b[0] = 0;
  }
  return __syncthreads_and(fits && (!seqs || (red[PG_MANY / 32].x <= limit_a && red[PG_MANY / 32].y <= limit_b)));
}

// The sequence s with sums[s] <= item < sums[s + 1].
RTR_DEVICE int page_seq(const int32_t* sums, int seqs, int item) {
  int lo = 0, hi = seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid + 1] > item) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// ROWS: rows a thread; with four, positions are one 16-byte store.
template <int ROWS>
__global__ void __launch_bounds__(PG_MANY) pages_grow_kernel(const PagePool p, const PageSeqs q, const int32_t* fresh,
                                                                int each, int rows, int32_t* lens, int32_t* starts_out,
                                                                int32_t* positions, int64_t* slots) {
  extern __shared__ int32_t pg_sums[];
  int32_t *starts = pg_sums, *items = pg_sums + q.seqs + 1;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, shift = p.shift, count = *p.count;
  const int64_t room = (int64_t)q.width << shift;
  const bool counted = count >= 0 && count <= p.pages;
  const auto value = [&](int s, int& n, int& need) {
    const int h = q.held[s];
    n = fresh ? fresh[s] : each;
    if (h < 0 || n < 0 || (int64_t)h + n > room) return false;
    need = pages_of(h + n, shift) - pages_of(h, shift);
    return true;
  };
  const bool fits = page_sums(q.seqs, starts, items, rows, INT32_MAX, value);
  const int all = fits ? items[q.seqs] : 0;
  const bool enough = counted && all <= count;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + tid, step = (int64_t)gridDim.x * blockDim.x;
  if (!fits || !enough) {
    if (at == 0) atomicOr(p.status, fits ? RTR_DEV_FEW_PAGES : RTR_DEV_BAD_LENGTH);
    for (int64_t s = at; s <= q.seqs; s += step) {
      starts_out[s] = 0;
      if (s < q.seqs) lens[s] = q.held[s];
    }
    for (int64_t r = at; r < rows; r += step) {
      positions[r] = -1;
      slots[r] = -1;
    }
    return;
  }
  for (int64_t s = at; s <= q.seqs; s += step) {
    starts_out[s] = starts[s];
    if (s < q.seqs) lens[s] = q.held[s] + starts[s + 1] - starts[s];
  }
  const int32_t* top = p.free + count - 1;
  for (int64_t i = at; i < all; i += step) {
    const int s = page_seq(items, q.seqs, (int)i), page = top[-i];
    q.table[s * q.stride + pages_of(q.held[s], shift) + (i - items[s])] = page;
    if (page >= 0 && page < p.pages) p.marks[page] = 1;
    else atomicOr(p.status, RTR_DEV_BAD_PAGE);
  }
  const int end = starts[q.seqs];
  for (int64_t r0 = at * ROWS; r0 < rows; r0 += step * ROWS) {
    // the rows' sequences, then all their loads at a time
    int32_t pos[ROWS], page[ROWS];
    int64_t slot[ROWS];
    int s = r0 < end ? page_seq(starts, q.seqs, (int)r0) : 0;
    const int32_t* from[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      from[j] = nullptr;
      pos[j] = -1;
      if (r0 + j >= end) continue;
      const int r = (int)r0 + j;
      while (starts[s + 1] <= r) ++s;
      const int had = q.held[s], t = had + r - starts[s], nth = t >> shift, old = pages_of(had, shift);
      pos[j] = t;
      from[j] = nth < old ? q.table + s * q.stride + nth : top - (int64_t)(items[s] + nth - old);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) page[j] = from[j] ? *from[j] : -1;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      slot[j] = -1;
      if (page[j] >= 0 && page[j] < p.pages) {
        slot[j] = ((int64_t)page[j] << shift) + (pos[j] & ((1 << shift) - 1));
      } else {
        if (from[j]) atomicOr(p.status, RTR_DEV_BAD_PAGE);
        pos[j] = -1;
      }
    }
    if (ROWS == 4 && r0 + ROWS <= rows) {
      *reinterpret_cast<int4*>(positions + r0) = make_int4(pos[0], pos[1 % ROWS], pos[2 % ROWS], pos[3 % ROWS]);
      *reinterpret_cast<longlong2*>(slots + r0) = make_longlong2(slot[0], slot[1 % ROWS]);
      *reinterpret_cast<longlong2*>(slots + r0 + 2) = make_longlong2(slot[2 % ROWS], slot[3 % ROWS]);
    } else {
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
        if (r0 + j < rows) {
          positions[r0 + j] = pos[j];
          slots[r0 + j] = slot[j];
        }
    }
  }
  // The stack's height changes when every block has read it.  (Nothing else of one block is read by another: no fence.)
  __syncthreads();
  if (tid == 0) {
    if (gridDim.x == 1) {
      *p.count = count - all;
    } else if (atomicAdd(p.ticket, 1u) == gridDim.x - 1) {
      *p.ticket = 0;
      *p.count = count - all;
    }
  }
}

__global__ void __launch_bounds__(PG_MANY) pages_release_kernel(const PagePool p, const PageSeqs q,
                                                                        const int32_t* keep) {
  extern __shared__ int32_t pg_sums[];
  __shared__ uint32_t wrong;
  pdl_launch_dependents();
  pdl_wait();
  const auto cluster = cooperative_groups::this_cluster();
  const int tid = threadIdx.x, shift = p.shift, count = *p.count;
  const int at = (int)cluster.block_rank() * blockDim.x + tid, step = (int)cluster.num_blocks() * blockDim.x;
  const int64_t room = (int64_t)q.width << shift;
  if (tid == 0) wrong = 0;
  const bool fits = page_sums(q.seqs, pg_sums, nullptr, INT32_MAX, INT32_MAX, [&](int s, int& n, int&) {
    const int h = q.held[s], k = keep ? keep[s] : 0;
    if (k < 0 || k > h || h > room) return false;
    n = pages_of(h, shift) - pages_of(k, shift);
    return true;
  });
  if (!fits) {  // every block of the cluster says the same
    if (at == 0) atomicOr(p.status, RTR_DEV_BAD_LENGTH);
    return;
  }
  const int all = pg_sums[q.seqs];
  // each thread has neighbouring items: one search, then from sequence to sequence
  const int share = (all - 1) / step + 1, lo = (int)min((int64_t)at * share, (int64_t)all), hi = (int)min((int64_t)lo + share, (int64_t)all);
  const auto each = [&](int from, auto&& f) {
    int s = from < hi ? page_seq(pg_sums, q.seqs, from) : 0;
    for (int i = from; i < hi; ++i) {
      while (pg_sums[s + 1] <= i) ++s;
      f(i, q.table + s * q.stride + pages_of(keep ? keep[s] : 0, shift) + (i - pg_sums[s]));
    }
  };
  uint32_t bad = count < 0 || count > p.pages || all > p.pages - count ? RTR_DEV_PAGE_NOT_HELD : 0u;
  int held[PG_HELD];  // the thread's first pages
#pragma unroll
  for (int j = 0; j < PG_HELD; ++j) held[j] = -1;
  const auto mark = [&](int page) {
    if (page < 0 || page >= p.pages) bad |= RTR_DEV_BAD_PAGE;
    else if (atomicCAS(p.marks + page, 1, 2) != 1) bad |= RTR_DEV_PAGE_NOT_HELD;
  };
  if (!bad) {
    const int32_t* where[PG_HELD];
    int s = lo < hi ? page_seq(pg_sums, q.seqs, lo) : 0;
#pragma unroll
    for (int j = 0; j < PG_HELD; ++j) {
      const int i = lo + j;
      if (i >= hi) break;
      while (pg_sums[s + 1] <= i) ++s;
      where[j] = q.table + s * q.stride + pages_of(keep ? keep[s] : 0, shift) + (i - pg_sums[s]);
    }
#pragma unroll
    for (int j = 0; j < PG_HELD; ++j)
      if (lo + j < hi) held[j] = *where[j];
#pragma unroll
    for (int j = 0; j < PG_HELD; ++j)
      if (lo + j < hi) mark(held[j]);
    each(lo + PG_HELD, [&](int, const int32_t* at_) { mark(*at_); });
  }
  if (bad) atomicOr(&wrong, bad);
  cluster.sync();
  bad = 0;
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) bad |= *cluster.map_shared_rank(&wrong, r);
  const auto settle = [&](int i, int page) {
    if (!bad) {
      p.marks[page] = 0;
      p.free[(int64_t)count + all - 1 - i] = page;
    } else if (page >= 0 && page < p.pages && p.marks[page] == 2) {
      p.marks[page] = 1;
    }
  };
#pragma unroll
  for (int j = 0; j < PG_HELD; ++j)
    if (lo + j < hi) settle(lo + j, held[j]);
  each(lo + PG_HELD, [&](int i, const int32_t* at_) { settle(i, *at_); });
  if (at == 0) {
    if (bad) atomicOr(p.status, bad);
    else *p.count = count + all;
  }
  cluster.sync();  // no block leaves while another may still read its word
}

static const char* pages_check(const rtr_page_pool* p, const void* table, int64_t stride, int32_t width, const void* held,
                               int32_t seqs) {
  if (!p || !p->free || !p->count || !p->marks || !p->status || !p->ticket) return "null pool or pool buffer";
  if (p->pages < 1) return "a pool needs pages";
  if (p->page < 1 || p->page > 1024 || (p->page & (p->page - 1))) return "page must be a power of two from 1 to 1024 tokens";
  if (seqs < 0 || seqs > PG_MAX_SEQS) return "0 to 16384 sequences in one call";
  if (seqs && (!table || !held)) return "null table or lengths";
  if (seqs && (width < 1 || stride < width)) return "table rows overlap or are empty";
  if ((int64_t)width * p->page > INT32_MAX - 4096) return "a table row holds at most 2^31 - 4096 tokens";
  return nullptr;
}

static PagePool device_pool(const rtr_page_pool* p) {
  int shift = 0;
  while ((1 << shift) < p->page) ++shift;
  return PagePool{p->free, p->count, p->marks, p->status, p->ticket, p->pages, shift};
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_pages_grow(const rtr_page_pool* pool, int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* held,
                   const int32_t* fresh, int32_t each, int32_t seqs, int32_t rows, int32_t* lens, int32_t* starts,
                   int32_t* positions, int64_t* slots, int32_t device, void* stream) {
  if (const char* e = pages_check(pool, table, table_stride, table_width, held, seqs)) return set_error(RTR_ERR_ARG, e);
  if (rows < 0 || each < 0) return set_error(RTR_ERR_ARG, "negative row or token count");
  if (!starts || (seqs && !lens) || (rows && (!positions || !slots))) return set_error(RTR_ERR_ARG, "null output");
  if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots)) & 15)
    return set_error(RTR_ERR_ARG, "positions and slots must lie at multiples of 16 bytes");
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  // A block for as many rows (four a thread where one each would be more blocks than fill the GPU) and sequences as it has threads, and
  // no more than fill the GPU four times: a block's own scan of the lengths is then a small part of what it does.
  const int threads = seqs <= PG_FEW ? PG_FEW : PG_MANY, room = on.sms * (2048 / threads);
  const bool four = rows > (int64_t)room * threads / 4;
  const int64_t each_block = (int64_t)threads * (four ? 4 : 1);
  const int64_t want = std::max<int64_t>((rows + each_block - 1) / each_block, (seqs + threads) / threads);
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(want, 1), 4 * (int64_t)room);
  const int smem = 2 * (seqs + 1) * (int)sizeof(int32_t), most = 2 * (PG_MAX_SEQS + 1) * (int)sizeof(int32_t);
  static std::atomic<uint64_t> allowed[2];
  const auto run = [&](auto kernel) {
    const cudaError_t e = smem > 32 << 10 ? kv_allow_smem(kernel, most, allowed[four], device) : cudaSuccess;
    return e != cudaSuccess ? e : kv_launch(kernel, dim3(grid), threads, smem, 1, static_cast<cudaStream_t>(stream), device_pool(pool),
                  PageSeqs{table, table_stride, table_width, seqs, held}, fresh, (int)each, (int)rows, lens, starts, positions,
                  slots);
  };
  const cudaError_t e = four ? run(pages_grow_kernel<4>) : run(pages_grow_kernel<1>);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

int rtr_pages_release(const rtr_page_pool* pool, const int32_t* table, int64_t table_stride, int32_t table_width,
                      const int32_t* held, const int32_t* keep, int32_t seqs, int32_t device, void* stream) {
  if (const char* e = pages_check(pool, table, table_stride, table_width, held, seqs)) return set_error(RTR_ERR_ARG, e);
  if (!seqs) return RTR_OK;
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  // How many pages come back is not known here, only the tables' entries: one block for two entries a thread, a cluster of up to eight
  // for more.  (64 x 66 entries, 64 pages at most given back and taken: one block 7.8 us, four 8.4, eight 9.4; 96 x 66, 4,000 pages: 14.9,
  // 10.5 and 10.5.)
  const int64_t entries = (int64_t)seqs * table_width;
  const int threads = entries <= 2 * PG_FEW ? PG_FEW : PG_MANY;
  int cluster = 1;
  while (cluster < PG_BACK_CLUSTER && entries > (int64_t)PG_PER * cluster * threads) cluster *= 2;
  const int smem = (seqs + 1) * (int)sizeof(int32_t);
  static std::atomic<uint64_t> allowed;
  cudaError_t e = smem > 32 << 10 ? kv_allow_smem(pages_release_kernel, (PG_MAX_SEQS + 1) * (int)sizeof(int32_t), allowed, device)
                                  : cudaSuccess;
  if (e == cudaSuccess)
    e = kv_launch(pages_release_kernel, dim3(1, 1, cluster), threads, smem, cluster, static_cast<cudaStream_t>(stream),
                  device_pool(pool), PageSeqs{const_cast<int32_t*>(table), table_stride, table_width, seqs, held}, keep);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
