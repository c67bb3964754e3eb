// Page numbers handed out and taken back on the GPU: page tables, row offsets, positions and
// slots from the lengths of a batch of sequences.
//
// Mathematics.  n tokens need ceil(n / page) pages.  With need[b] = pages(held + fresh) - pages(held)
// the call's page items are numbered by the running sum of need, its rows by the running
// sum of fresh; item j takes the j-th number from the top of the stack of free pages.  Everything else is a search of an item
// or a row in those two sums.
//
// What bounds it.  Some kilobytes for a step's tokens: the launch and three dependent loads (lengths,
// table or stack, store), with the block's scan between them.  For prompts the 12 bytes a
// row are written at L2's rate.  So one launch does it all: every block sums the lengths itself
// (they are in L2, and a scan of 2,000 sequences costs less than a second launch or a barrier
// over the grid) and then takes its share of rows and items.  A call that does not fit must
// change nothing, and every block finds that out for itself from the same numbers.
// Taking changes the stack's height alone, which the last block to finish does, by a ticket; a page
// item of the call is read from the stack by whoever needs it, so no block waits for another.
//
// Giving back is all or nothing over values that lie in the table (a page number that is out of
// range, or that no sequence holds), so its blocks have to agree before any of them writes: they are
// one cluster, which marks every page first, then pushes them or takes the marks back.
#include <cuda_runtime.h>

#include <cooperative_groups.h>

#include "engine.h"
#include "kv_host.h"

namespace rtr {

constexpr int PG_THREADS = 256, PG_MAX_SEQS = 16384, PG_ROWS = 4;  // rows a thread: one 16-byte store of positions
constexpr int PG_BACK_THREADS = 512, PG_BACK_CLUSTER = 8;

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

RTR_DEVICE int pages_of(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

// The running sums of two numbers a sequence, by all threads of the block: a[0 .. seqs], b[0 .. seqs]
// (b null: one number).  value(s, x, y) gives sequence s's two numbers and false where it does not fit; the
// result is false where any sequence does not fit or a sum is above its limit.  Each thread takes consecutive sequences.
template <typename F>
RTR_DEVICE bool page_sums(int seqs, int32_t* a, int32_t* b, int64_t* red, int64_t limit_a, int64_t limit_b, F&& value) {
  const int tid = threadIdx.x, warps = blockDim.x >> 5, lane = tid & 31, warp = tid >> 5;
  const int per = (seqs + blockDim.x - 1) / blockDim.x, lo = min(seqs, tid * per), hi = min(seqs, lo + per);
  int64_t x = 0, y = 0;
  int fits = 1;
  for (int s = lo; s < hi; ++s) {
    int p = 0, q = 0;
    if (!value(s, p, q)) fits = p = q = 0;
    a[s + 1] = p;
    if (b) b[s + 1] = q;
    x += p;
    y += q;
  }
  int64_t xs = x, ys = y;  // inclusive over the warp
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, xs, d), v = __shfl_up_sync(0xffffffffu, ys, d);
    if (lane >= d) {
      xs += u;
      ys += v;
    }
  }
  if (lane == 31) {
    red[2 * warp] = xs;
    red[2 * warp + 1] = ys;
  }
  fits = __syncthreads_and(fits);
  int64_t all_x = 0, all_y = 0;
  for (int w = 0; w < warps; ++w) {
    if (w == warp) {
      xs += all_x;
      ys += all_y;
    }
    all_x += red[2 * w];
    all_y += red[2 * w + 1];
  }
  const bool good = fits && all_x <= limit_a && all_y <= limit_b;
  if (good) {  // the sums fit 32 bits: limits do
    xs -= x;
    ys -= y;
    if (tid == 0) {
      a[0] = 0;
      if (b) b[0] = 0;
    }
    for (int s = lo; s < hi; ++s) {
      xs += a[s + 1];
      a[s + 1] = (int32_t)xs;
      if (b) {
        ys += b[s + 1];
        b[s + 1] = (int32_t)ys;
      }
    }
  }
  __syncthreads();
  return good;
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

__global__ void __launch_bounds__(PG_THREADS) pages_grow_kernel(const PagePool p, const PageSeqs q, const int32_t* fresh,
                                                                int each, int rows, int32_t* lens, int32_t* starts_out,
                                                                int32_t* positions, int64_t* slots) {
  extern __shared__ int32_t pg_sums[];
  __shared__ int64_t red[2 * PG_THREADS / 32];
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
  const bool fits = page_sums(q.seqs, starts, items, red, rows, INT32_MAX, value);
  const int all = fits ? items[q.seqs] : 0;
  const bool enough = counted && all <= count;
  const int64_t at = (int64_t)blockIdx.x * PG_THREADS + tid, step = (int64_t)gridDim.x * PG_THREADS;
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
  for (int64_t r0 = at * PG_ROWS; r0 < rows; r0 += step * PG_ROWS) {
    int32_t pos[PG_ROWS];
    int64_t slot[PG_ROWS];
    int s = r0 < end ? page_seq(starts, q.seqs, (int)r0) : 0, had = -1, of = -1, nth = -1, page = -1;
#pragma unroll
    for (int j = 0; j < PG_ROWS; ++j) {
      const int r = (int)min(r0 + j, (int64_t)INT32_MAX);
      pos[j] = -1;
      slot[j] = -1;
      if (r >= end) continue;
      while (starts[s + 1] <= r) ++s;
      if (s != of) {
        had = q.held[s];
        of = s;
        nth = -1;
      }
      const int t = had + r - starts[s];
      if (t >> shift != nth) {
        nth = t >> shift;
        const int old = pages_of(had, shift);
        page = nth < old ? q.table[s * q.stride + nth] : top[-(int64_t)(items[s] + nth - old)];
        if (page < 0 || page >= p.pages) {
          atomicOr(p.status, RTR_DEV_BAD_PAGE);
          page = -1;
        }
      }
      if (page >= 0) {
        pos[j] = t;
        slot[j] = ((int64_t)page << shift) + (t & ((1 << shift) - 1));
      }
    }
    if (r0 + PG_ROWS <= rows) {
      *reinterpret_cast<int4*>(positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(slots + r0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(slots + r0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int j = 0; j < PG_ROWS; ++j)
        if (r0 + j < rows) {
          positions[r0 + j] = pos[j];
          slots[r0 + j] = slot[j];
        }
    }
  }
  // The stack's height changes when every block has read it (and what lies below it).
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    if (atomicAdd(p.ticket, 1u) == gridDim.x - 1) {
      *p.ticket = 0;
      *p.count = count - all;
    }
  }
}

__global__ void __launch_bounds__(PG_BACK_THREADS) pages_release_kernel(const PagePool p, const PageSeqs q,
                                                                        const int32_t* keep) {
  extern __shared__ int32_t pg_sums[];
  __shared__ int64_t red[2 * PG_BACK_THREADS / 32];
  __shared__ uint32_t wrong;
  pdl_launch_dependents();
  pdl_wait();
  const auto cluster = cooperative_groups::this_cluster();
  const int tid = threadIdx.x, shift = p.shift, count = *p.count;
  const int at = (int)cluster.block_rank() * PG_BACK_THREADS + tid, step = (int)cluster.num_blocks() * PG_BACK_THREADS;
  const int64_t room = (int64_t)q.width << shift;
  if (tid == 0) wrong = 0;
  const bool fits = page_sums(q.seqs, pg_sums, nullptr, red, INT32_MAX, INT32_MAX, [&](int s, int& n, int&) {
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
  const auto page_at = [&](int i) {
    const int s = page_seq(pg_sums, q.seqs, i), k = keep ? keep[s] : 0;
    return q.table[s * q.stride + pages_of(k, shift) + (i - pg_sums[s])];
  };
  uint32_t bad = count < 0 || count > p.pages || all > p.pages - count ? RTR_DEV_PAGE_NOT_HELD : 0u;
  if (!bad) {
    for (int64_t i = at; i < all; i += step) {
      const int page = page_at((int)i);
      if (page < 0 || page >= p.pages) bad |= RTR_DEV_BAD_PAGE;
      else if (atomicCAS(p.marks + page, 1, 2) != 1) bad |= RTR_DEV_PAGE_NOT_HELD;
    }
  }
  if (bad) atomicOr(&wrong, bad);
  cluster.sync();
  bad = 0;
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) bad |= *cluster.map_shared_rank(&wrong, r);
  for (int64_t i = at; i < all; i += step) {
    const int page = page_at((int)i);
    if (!bad) {
      p.marks[page] = 0;
      p.free[(int64_t)count + all - 1 - i] = page;
    } else if (page >= 0 && page < p.pages && p.marks[page] == 2) {
      p.marks[page] = 1;
    }
  }
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
  // A block for every 1,024 rows, every 256 sequences, and no more than fill the GPU four times: a
  // block's own scan of the lengths is then a small part of what it does.
  const int64_t want = std::max<int64_t>((rows + PG_THREADS * PG_ROWS - 1) / (PG_THREADS * PG_ROWS), (seqs + PG_THREADS) / PG_THREADS);
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(want, 1), 4 * (int64_t)on.sms);
  const int smem = 2 * (seqs + 1) * (int)sizeof(int32_t);
  static std::atomic<uint64_t> allowed;
  cudaError_t e = smem > 32 << 10 ? kv_allow_smem(pages_grow_kernel, 2 * (PG_MAX_SEQS + 1) * (int)sizeof(int32_t), allowed, device)
                                  : cudaSuccess;
  if (e == cudaSuccess)
    e = kv_launch(pages_grow_kernel, dim3(grid), PG_THREADS, smem, 1, static_cast<cudaStream_t>(stream), device_pool(pool),
                  PageSeqs{table, table_stride, table_width, seqs, held}, fresh, (int)each, (int)rows, lens, starts, positions,
                  slots);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

int rtr_pages_release(const rtr_page_pool* pool, const int32_t* table, int64_t table_stride, int32_t table_width,
                      const int32_t* held, const int32_t* keep, int32_t seqs, int32_t device, void* stream) {
  if (const char* e = pages_check(pool, table, table_stride, table_width, held, seqs)) return set_error(RTR_ERR_ARG, e);
  if (!seqs) return RTR_OK;
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  // One block while every page that the tables can name is a round of its threads or two.
  const int cluster = (int64_t)seqs * table_width <= 2 * PG_BACK_THREADS ? 1 : PG_BACK_CLUSTER;
  const int smem = (seqs + 1) * (int)sizeof(int32_t);
  static std::atomic<uint64_t> allowed;
  cudaError_t e = smem > 32 << 10 ? kv_allow_smem(pages_release_kernel, (PG_MAX_SEQS + 1) * (int)sizeof(int32_t), allowed, device)
                                  : cudaSuccess;
  if (e == cudaSuccess)
    e = kv_launch(pages_release_kernel, dim3(1, 1, cluster), PG_BACK_THREADS, smem, cluster, static_cast<cudaStream_t>(stream),
                  device_pool(pool), PageSeqs{const_cast<int32_t*>(table), table_stride, table_width, seqs, held}, keep);
  return e == cudaSuccess ? RTR_OK : set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
