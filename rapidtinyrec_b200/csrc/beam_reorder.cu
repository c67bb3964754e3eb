// The beams' states put in the order of their parents, in place, many tensors in one launch.
//
// A column is 16 bytes of a row (4 or 1 where the states do not lie at multiples of 16) and the same bytes of the item's other
// beams.  One thread moves one: it brings every row that is a parent of another beam into shared memory by asynchronous
// copies, waits for its own alone, and writes the rows that change.  Nobody else touches the column,
// so there is no second buffer, no barrier and no order among blocks; rows that stay are neither read
// nor written, a parent of many children is read once.
//
// What bounds it: HBM (L2 where the states fit).  50 rows of 64 columns are 51 KB, four blocks an SM have up to 200 KB in
// flight.  A block goes over several tiles of columns with one look at the parents.  576 MB moved (400 rows, 28 states): 98.4 us, 5.9
// TB/s, 90 % of the copy rate; 8.5 MB of one item, in L2: 7 us, of which launch, parents, rows in and rows out are a chain of four waits.
#include <cuda_runtime.h>

#include "engine.h"
#include "kv_host.h"

namespace rtr {

constexpr int BR_THREADS = 64, BR_MAX_BEAMS = 128, BR_STATES = 32;  // states of one launch: their layouts are its arguments

struct MoveState {
  char* data;
  int64_t row, strides[3];
  uint32_t sizes[3], inner;  // inner: columns
  uint32_t tile0, columns;   // first tile of the launch, columns of a row
};
struct Moves {
  MoveState states[BR_STATES];
  const int32_t* parents;
  uint32_t* status;
  int count, beams, per;  // per: columns a thread has in flight
  uint32_t tiles;
};

template <int VEC> RTR_DEVICE void move_in(char* to, const char* from) {
  if constexpr (VEC == 16) {
    cp_async16(to, from, true);
  } else if constexpr (VEC == 4) {
    const unsigned s = static_cast<unsigned>(__cvta_generic_to_shared(to));
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(s), "l"(from));
  } else {
    *to = *from;
  }
}
template <int VEC> RTR_DEVICE void move_out(char* to, const char* from) {
  if constexpr (VEC == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
  else *to = *from;
}

template <int VEC>
__global__ void __launch_bounds__(BR_THREADS) beam_reorder_kernel(const __grid_constant__ Moves m) {
  extern __shared__ __align__(16) char br_rows[];
  __shared__ uint32_t read[BR_MAX_BEAMS / 32], moved[BR_MAX_BEAMS / 32];
  __shared__ uint8_t from[BR_MAX_BEAMS];                      // rows that are read, by their slot
  __shared__ uint8_t to[BR_MAX_BEAMS], slot[BR_MAX_BEAMS];    // rows that are written, and the slots of their parents
  const int tid = threadIdx.x, item = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  if (tid < BR_MAX_BEAMS / 32) read[tid] = moved[tid] = 0;
  __syncthreads();
  int parent[BR_MAX_BEAMS / BR_THREADS];
#pragma unroll
  for (int j = 0; j < BR_MAX_BEAMS / BR_THREADS; ++j) {
    const int i = tid + j * BR_THREADS;
    parent[j] = i;
    if (i < m.beams) {
      const int p = m.parents[(int64_t)item * m.beams + i];
      if (p < 0 || p >= m.beams) {
        if (blockIdx.x == 0) atomicOr(m.status, RTR_DEV_BAD_PARENT);
      } else if (p != i) {
        parent[j] = p;
        atomicOr(&read[p >> 5], 1u << (p & 31));
        atomicOr(&moved[i >> 5], 1u << (i & 31));
      }
    }
  }
  __syncthreads();
  const auto place = [](const uint32_t (&bits)[BR_MAX_BEAMS / 32], int i) {  // how many are set before bit i
    int n = __popc(bits[i >> 5] & ((1u << (i & 31)) - 1));
    for (int w = 0; w < i >> 5; ++w) n += __popc(bits[w]);
    return n;
  };
  int reads = 0, writes = 0;
#pragma unroll
  for (int w = 0; w < BR_MAX_BEAMS / 32; ++w) {
    reads += __popc(read[w]);
    writes += __popc(moved[w]);
  }
#pragma unroll
  for (int j = 0; j < BR_MAX_BEAMS / BR_THREADS; ++j) {
    const int i = tid + j * BR_THREADS;
    if (read[i >> 5] >> (i & 31) & 1) from[place(read, i)] = (uint8_t)i;
    if (parent[j] != i) {
      const int d = place(moved, i);
      to[d] = (uint8_t)i;
      slot[d] = (uint8_t)place(read, parent[j]);
    }
  }
  __syncthreads();
  if (!writes) return;
  char* mine = br_rows + tid * VEC;
  int s = 0;
  for (uint32_t tile = blockIdx.x; tile < m.tiles; tile += gridDim.x) {
    while (s + 1 < m.count && m.states[s + 1].tile0 <= tile) ++s;
    const MoveState& st = m.states[s];
    char* at[8];
    for (int j = 0; j < m.per; ++j) {
      const uint32_t column = ((tile - st.tile0) * m.per + j) * BR_THREADS + tid;
      at[j & 7] = nullptr;
      if (column >= st.columns) continue;
      const uint32_t o = column / st.inner, o2 = o / st.sizes[2], o1 = o2 / st.sizes[1];
      char* p = st.data + (int64_t)item * m.beams * st.row + (int64_t)(column - o * st.inner) * VEC +
                (int64_t)(o - o2 * st.sizes[2]) * st.strides[2] + (int64_t)(o2 - o1 * st.sizes[1]) * st.strides[1] +
                (int64_t)o1 * st.strides[0];
      at[j & 7] = p;
      for (int r = 0; r < reads; ++r) move_in<VEC>(mine + (j * reads + r) * (BR_THREADS * VEC), p + from[r] * st.row);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();  // keeps the compiler from reading the rows before they are there
    for (int j = 0; j < m.per; ++j) {
      char* p = at[j & 7];
      if (!p) continue;
#pragma unroll 4
      for (int d = 0; d < writes; ++d) move_out<VEC>(p + to[d] * st.row, mine + (j * reads + slot[d]) * (BR_THREADS * VEC));
    }
    __syncwarp();  // or writing the next tile's before these are read
  }
}

// Bytes of a column: 16 or 4 where all of a state lies at multiples of them, else 1.
static int state_column(const rtr_beam_state& s) {
  uint64_t bits = reinterpret_cast<uintptr_t>(s.data) | (uint64_t)s.row_bytes | (uint64_t)s.inner;
  for (int d = 0; d < 3; ++d)
    if (s.sizes[d] > 1) bits |= (uint64_t)s.strides[d];
  return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
}
static const char* state_check(const rtr_beam_state& s) {
  if (!s.data) return "null state";
  if (s.inner < 1 || s.sizes[0] < 1 || s.sizes[1] < 1 || s.sizes[2] < 1) return "a state's dimensions must be positive";
  if (s.row_bytes == 0) return "the rows of a state overlap";
  for (int d = 0; d < 3; ++d)
    if (s.sizes[d] > 1 && s.strides[d] == 0) return "a state's dimensions overlap";
  uint64_t columns = (uint64_t)s.inner / state_column(s);
  for (int d = 0; d < 3 && columns <= INT32_MAX; ++d) columns *= (uint64_t)s.sizes[d];
  return columns > INT32_MAX ? "a state's rows are too long" : nullptr;
}

}  // namespace rtr

using namespace rtr;

extern "C" {

int rtr_beam_reorder(const rtr_beam_state* states, int32_t count, const int32_t* parents, int32_t items, int32_t beams,
                     uint32_t* status, int32_t device, void* stream) {
  if (count < 0 || items < 0 || beams < 1 || beams > BR_MAX_BEAMS) return set_error(RTR_ERR_ARG, "0 or more states and items, 1 to 128 beams");
  if (items > 65535) return set_error(RTR_ERR_ARG, "at most 65535 items in one call");
  if (!count || !items) return RTR_OK;
  if (!states || !parents || !status) return set_error(RTR_ERR_ARG, "null states, parents or status");
  for (int i = 0; i < count; ++i)
    if (const char* e = state_check(states[i])) return set_error(RTR_ERR_ARG, e);
  KvDevice on(device);
  if (on.error) return set_error(RTR_ERR_CUDA, cudaGetErrorString(on.error));
  static std::atomic<uint64_t> allowed[3];
  for (int kind = 0; kind < 3; ++kind) {  // states at multiples of 16 bytes, of 4, and any others
    const int vec = kind == 0 ? 16 : kind == 1 ? 4 : 1;
    Moves m = {};
    m.parents = parents;
    m.status = status;
    m.beams = beams;
    // Eight rows or more in flight a thread: with few beams several columns of them (4 beams of 4 items, 59 MB moved: 4, 8, 16, 32 rows
    // 17.4, 13.3, 13.9, 22.3 us).
    m.per = std::max(1, 8 / beams);
    const uint64_t tile = (uint64_t)m.per * BR_THREADS;
    uint64_t tiles = 0;
    const auto launch = [&]() -> cudaError_t {
      const int smem = m.per * beams * BR_THREADS * vec, most = BR_MAX_BEAMS * BR_THREADS * vec;
      m.tiles = (uint32_t)tiles;
      // Eight times as many blocks as the SMs hold: a block's look at the parents is a small part of it, and so is the last
      // wave (400 rows of 1.4 MB: 1, 4, 8, 16 times 105.9, 102.2, 98.4, 101.8 us).
      const uint64_t fit = std::max(1, std::min(24, (227 << 10) / (smem + 1024)));
      const uint64_t want = std::max<uint64_t>(1, (8 * fit * (uint64_t)on.sms + items - 1) / items);
      const dim3 grid((unsigned)std::min<uint64_t>(tiles, want), (unsigned)items);
      const auto run = [&](auto kernel) {
        cudaError_t e = smem > 32 << 10 ? kv_allow_smem(kernel, most, allowed[kind], device) : cudaSuccess;
        return e == cudaSuccess ? kv_launch(kernel, grid, BR_THREADS, smem, 1, static_cast<cudaStream_t>(stream), m) : e;
      };
      const cudaError_t e = kind == 0 ? run(beam_reorder_kernel<16>) : kind == 1 ? run(beam_reorder_kernel<4>) : run(beam_reorder_kernel<1>);
      m.count = 0;
      tiles = 0;
      return e;
    };
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < count && e == cudaSuccess; ++i) {
      const rtr_beam_state& s = states[i];
      if (state_column(s) != vec) continue;
      const uint64_t inner = (uint64_t)s.inner / vec;
      const uint64_t columns = inner * s.sizes[0] * s.sizes[1] * s.sizes[2];
      const uint64_t more = (columns + tile - 1) / tile;
      if (m.count == BR_STATES || tiles + more > INT32_MAX) e = launch();
      MoveState& to = m.states[m.count++];
      to.data = static_cast<char*>(s.data);
      to.row = s.row_bytes;
      for (int d = 0; d < 3; ++d) {
        to.strides[d] = s.strides[d];
        to.sizes[d] = (uint32_t)s.sizes[d];
      }
      to.inner = (uint32_t)inner;
      to.columns = (uint32_t)columns;
      to.tile0 = (uint32_t)tiles;
      tiles += more;
    }
    if (e == cudaSuccess && m.count) e = launch();
    if (e != cudaSuccess) return set_error(RTR_ERR_CUDA, cudaGetErrorString(e));
  }
  return RTR_OK;
}

}  // extern "C"
