// The Python calls of the page pool (page_pool.py), rotary positions (rotary.py) and beam search
// (beam_search.py): argument checks, outputs and workspaces from torch's allocator, and one
// call into the C ABI each.  A handle's Python object keeps its C struct; a call gets its address.
#include "call.h"

#include <algorithm>
#include <vector>

namespace {

decltype(&rtr_pages_grow) pages_grow;
decltype(&rtr_pages_release) pages_release;
decltype(&rtr_rotary) rotary;
decltype(&rtr_beam_select_workspace) beam_workspace;
decltype(&rtr_beam_select) beam_select;
decltype(&rtr_beam_reorder) beam_reorder;

int64_t whole(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s must be an integer", name);
  }
  return v;
}

// What a call works on: the handle's C struct and its device.
template <typename T> struct Handle {
  const T* c;
  int index;
  Handle(PyObject* at, PyObject* device)
      : c(static_cast<const T*>(PyLong_AsVoidPtr(at))), index((int)PyLong_AsLong(device)) {
    if (PyErr_Occurred()) throw Raised{};
  }
};
void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
bool here(const at::Tensor& t, int index) { return t.is_cuda() && t.get_device() == index; }
at::Tensor room_for(int index, at::IntArrayRef size, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (c10::DeviceIndex)index), std::nullopt));
}
// Several new tensors in one piece of memory, 16 bytes apart at least: a call to the allocator costs a microsecond, a tensor of
// memory that is there a quarter of one.
struct Room {
  at::Tensor all;
  int64_t used = 0;
  Room(int index, int64_t bytes) : all(room_for(index, {bytes}, at::kByte)) {}
  static int64_t of(int64_t values, int64_t size) { return (values * size + 15) & ~(int64_t)15; }
  at::Tensor take(at::IntArrayRef size, at::ScalarType type) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                            c10::scalarTypeToTypeMeta(type));
    c10::TensorImpl* impl = t.unsafeGetTensorImpl();
    impl->set_sizes_contiguous(size);
    const int64_t each = c10::elementSize(type);
    impl->set_storage_offset(used / each);
    used += of(impl->numel(), each);
    return t;
  }
};
PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* t = PyTuple_New((Py_ssize_t)tensors.size());
  if (!t) throw Raised{};
  Py_ssize_t i = 0;
  for (const at::Tensor& x : tensors) PyTuple_SET_ITEM(t, i++, x.defined() ? THPVariable_Wrap(x) : Py_NewRef(Py_None));
  return t;
}
// A tensor that is written in place: none that autograd would want back as it was.
void written(const at::Tensor& t, const char* name) {
  if (t.requires_grad()) refuse("%s must not require a gradient", name);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int32_t type_of(const at::Tensor& x) { return x.scalar_type() == at::kFloat ? RTR_DTYPE_F32 : RTR_DTYPE_BF16; }

// ------------------------------------------------------------------ page pool
struct Seqs {
  at::Tensor table, held;
  int64_t seqs, width, stride;
};

const int32_t* counts_of(PyObject* o, int64_t seqs, int index, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != seqs || !t.is_contiguous() || !here(t, index))
    refuse("%s must be int32 [seqs], contiguous, on the pool's device", name);
  return static_cast<const int32_t*>(t.data_ptr());
}

Seqs seqs_of(PyObject* table_, PyObject* held_, int index) {
  Seqs s{tensor(table_, "table"), tensor(held_, "held"), 0, 0, 0};
  if (s.table.scalar_type() != at::kInt || s.table.dim() != 2) refuse("table must be int32 [seqs, width]");
  s.seqs = s.table.size(0);
  s.width = s.table.size(1);
  if (s.seqs > INT32_MAX || s.width > INT32_MAX) refuse("seqs and width must fit 32 bits");
  if (s.width > 1 && s.table.stride(1) != 1) refuse("the rows of table must be contiguous");
  if (s.seqs > 1 && s.table.stride(0) < s.width) refuse("the rows of table overlap");
  if (!here(s.table, index)) refuse("table must lie on the pool's device");
  s.stride = s.seqs > 1 ? s.table.stride(0) : s.width;
  counts_of(held_, s.seqs, index, "held");
  return s;
}

// grow(pool, device, table, held, fresh (int or tensor), rows or None)
PyObject* call_grow(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const Handle<rtr_page_pool> pool(a[0], a[1]);
    const Seqs s = seqs_of(a[2], a[3], pool.index);
    const int32_t* fresh = nullptr;
    int64_t each = 0, rows = 0;
    if (THPVariable_Check(a[4])) {
      fresh = counts_of(a[4], s.seqs, pool.index, "new");
      if (a[5] == Py_None) refuse("rows must be given where new is a tensor");
    } else {
      each = whole(a[4], "new");
      if (each < 0 || each > INT32_MAX) refuse("new must not be negative and must fit 32 bits");
      if (s.seqs && each > INT32_MAX / s.seqs) refuse("rows must fit 32 bits");
      rows = each * s.seqs;
    }
    if (a[5] != Py_None) rows = whole(a[5], "rows");
    if (rows < 0 || rows > INT32_MAX) refuse("rows must not be negative and must fit 32 bits");
    written(s.table, "table");
    Room out(pool.index, Room::of(s.seqs, 4) + Room::of(s.seqs + 1, 4) + Room::of(rows, 4) + Room::of(rows, 8));
    const at::Tensor lens = out.take({s.seqs}, at::kInt), starts = out.take({s.seqs + 1}, at::kInt),
                     positions = out.take({rows}, at::kInt), slots = out.take({rows}, at::kLong);
    check(pages_grow(pool.c, static_cast<int32_t*>(s.table.data_ptr()), s.stride, (int32_t)s.width,
                     static_cast<const int32_t*>(s.held.data_ptr()), fresh, (int32_t)each, (int32_t)s.seqs, (int32_t)rows,
                     static_cast<int32_t*>(lens.data_ptr()), static_cast<int32_t*>(starts.data_ptr()),
                     static_cast<int32_t*>(positions.data_ptr()), static_cast<int64_t*>(slots.data_ptr()), pool.index,
                     stream_of(pool.index)));
    return tuple_of({lens, starts, positions, slots});
  });
}

// release(pool, device, table, held, keep or None)
PyObject* call_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const Handle<rtr_page_pool> pool(a[0], a[1]);
    const Seqs s = seqs_of(a[2], a[3], pool.index);
    const int32_t* keep = a[4] == Py_None ? nullptr : counts_of(a[4], s.seqs, pool.index, "keep");
    check(pages_release(pool.c, static_cast<const int32_t*>(s.table.data_ptr()), s.stride, (int32_t)s.width,
                        static_cast<const int32_t*>(s.held.data_ptr()), keep, (int32_t)s.seqs, pool.index,
                        stream_of(pool.index)));
    Py_RETURN_NONE;
  });
}

// --------------------------------------------------------------------- rotary
// Where a tensor [rows, heads, dim] lies in memory: bytes from the first to behind the last.
std::pair<uintptr_t, uintptr_t> extent(const at::Tensor& t) {
  uintptr_t end = 1;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (!t.size(d)) return {0, 0};
    end += (uintptr_t)((t.size(d) - 1) * t.stride(d));
  }
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {at, at + end * t.element_size()};
}

// Whether two tensors of rows of heads x dim values, in memory they may share with others' rows, have a value in common
// (where their rows have one distance, the places within it decide; otherwise their extents do).
bool share(const at::Tensor& x, const at::Tensor& y) {
  const auto [x0, x1] = extent(x);
  const auto [y0, y1] = extent(y);
  if (x1 <= y0 || y1 <= x0) return false;
  const int64_t size = x.element_size();
  if (x.size(0) < 2 || y.size(0) < 2 || x.stride(0) != y.stride(0) || x.element_size() != y.element_size()) return true;
  const int64_t step = x.stride(0) * size;
  const int64_t wx = (int64_t)(x1 - x0) - (x.size(0) - 1) * step, wy = (int64_t)(y1 - y0) - (y.size(0) - 1) * step;
  const int64_t from = (((int64_t)(y0 - x0) % step) + step) % step;  // y's rows start this far behind one of x's
  return !(from >= wx && from + wy <= step);
}

bool same_rows(const at::Tensor& x, const at::Tensor& y) {
  if (x.data_ptr() != y.data_ptr()) return false;
  for (int d = 0; d < 3; ++d)
    if (x.size(d) > 1 && x.stride(d) != y.stride(d)) return false;
  return true;
}

void fill_rows(rtr_rotary_rows& r, const at::Tensor& in, const at::Tensor& out) {
  r.in = in.data_ptr();
  r.out = out.data_ptr();
  r.in_row = in.stride(0);
  r.in_head = in.stride(1);
  r.out_row = out.stride(0);
  r.out_head = out.stride(1);
  r.heads = (int32_t)in.size(1);
  // the stride of a dimension with one entry means nothing
  if (in.size(1) == 1) r.in_head = r.out_head = in.size(2);
  if (in.size(0) == 1) r.in_row = r.out_row = in.size(1) * in.size(2);
}

// rotate(turns, head_dim, rotary_dim, interleaved, factor, q, k or None, positions, back, out or None)
PyObject* call_rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const at::Tensor& turns = tensor(a[0], "turns");
    const int index = turns.get_device();
    const int64_t dim = whole(a[1], "head_dim"), part = whole(a[2], "rotary_dim");
    const int interleaved = PyObject_IsTrue(a[3]), back = PyObject_IsTrue(a[8]);
    const double factor = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) throw Raised{};
    const bool two = a[6] != Py_None;
    at::Tensor in[2], out[2];
    in[0] = tensor(a[5], "q");
    if (two) in[1] = tensor(a[6], "k");
    const char* names[2] = {"q", "k"};
    const int64_t rows = in[0].dim() ? in[0].size(0) : 0;
    for (int i = 0; i < 1 + two; ++i) {
      if (in[i].dim() != 3 || in[i].size(0) != rows || in[i].size(1) < 1 || in[i].size(2) != dim || !here(in[i], index))
        refuse("%s must be [rows, heads, %lld] on the handle's device", names[i], (long long)dim);
      if (in[i].scalar_type() != at::kFloat && in[i].scalar_type() != at::kBFloat16)
        refuse("%s must be float32 or bfloat16", names[i]);
      if (in[i].scalar_type() != in[0].scalar_type()) refuse("q and k must have one type");
      if (in[i].size(1) > INT32_MAX / 2) refuse("too many heads");
    }
    const at::Tensor& positions = tensor(a[7], "positions");
    if ((positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong) || positions.dim() != 1 ||
        positions.size(0) != rows || !positions.is_contiguous() || !here(positions, index))
      refuse("positions must be int32 or int64 [rows], contiguous, on the handle's device");
    if (a[9] == Py_None) {
      for (int i = 0; i < 1 + two; ++i) {
        if (in[i].stride(2) != 1) in[i] = in[i].clone(at::MemoryFormat::Contiguous);
        out[i] = room_for(index, in[i].sizes(), in[i].scalar_type());
      }
    } else {
      if (two) {
        if ((!PyTuple_Check(a[9]) && !PyList_Check(a[9])) || PySequence_Fast_GET_SIZE(a[9]) != 2) refuse("out must be a pair of tensors");
        out[0] = tensor(PySequence_Fast_GET_ITEM(a[9], 0), "out");
        out[1] = tensor(PySequence_Fast_GET_ITEM(a[9], 1), "out");
      } else {
        out[0] = tensor(a[9], "out");
      }
      for (int i = 0; i < 1 + two; ++i) {
        const at::Tensor& o = out[i];
        if (o.sizes() != in[i].sizes() || o.scalar_type() != in[i].scalar_type() || !here(o, index) || o.stride(2) != 1)
          refuse("out must be like %s, its dimensions contiguous", names[i]);
        if ((rows > 1 && o.stride(0) < dim) || (o.size(1) > 1 && o.stride(1) < dim) ||
            (rows > 1 && o.size(1) > 1 && o.stride(0) < (o.size(1) - 1) * o.stride(1) + dim && o.stride(1) < (rows - 1) * o.stride(0) + dim))
          refuse("the rows of out overlap");
        if (!same_rows(o, in[i])) {
          if (share(o, in[i])) refuse("out must be %s itself or lie apart from it", names[i]);
          if (in[i].stride(2) != 1) in[i] = in[i].clone(at::MemoryFormat::Contiguous);
        }
      }
      if (two && rows && (share(out[0], out[1]) || share(out[0], in[1]) || share(out[1], in[0])))
        refuse("out of q and of k must not share memory with one another or the other's input");
    }
    if (a[9] != Py_None)
      for (int i = 0; i < 1 + two; ++i) written(out[i], "out");
    rtr_rotary_rows q = {}, k = {};
    fill_rows(q, in[0], out[0]);
    if (two) fill_rows(k, in[1], out[1]);
    check(rotary(&q, two ? &k : nullptr, rows, (int32_t)dim, (int32_t)part, interleaved, type_of(in[0]), positions.data_ptr(),
                 positions.scalar_type() == at::kLong, static_cast<const uint64_t*>(turns.data_ptr()), (float)factor, back, index,
                 stream_of(index)));
    if (!two) return THPVariable_Wrap(out[0]);
    return tuple_of({out[0], out[1]});
  });
}

// ---------------------------------------------------------------- beam search
// select(status address, device, beams, eos or None, candidates, logits, scores, allowed or None)
PyObject* call_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    uint32_t* status = static_cast<uint32_t*>(PyLong_AsVoidPtr(a[0]));
    const int index = (int)PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) throw Raised{};
    const int64_t beams = whole(a[2], "beams"), eos = a[3] == Py_None ? -1 : whole(a[3], "eos"), k = whole(a[4], "candidates");
    at::Tensor logits = tensor(a[5], "logits"), scores = tensor(a[6], "scores");
    if (logits.dim() != 2 || (logits.scalar_type() != at::kFloat && logits.scalar_type() != at::kBFloat16) || !here(logits, index))
      refuse("logits must be float32 or bfloat16 [items * beams, vocab] on the handle's device");
    if (scores.dim() != 2 || scores.scalar_type() != at::kFloat || !scores.is_contiguous() || !here(scores, index))
      refuse("scores must be float32 [items, beams], contiguous, on the handle's device");
    const int64_t items = scores.size(0), width = scores.size(1), rows = logits.size(0), vocab = logits.size(1);
    if (width < 1 || width > 128) refuse("1 to 128 beams an item");
    if (rows != items * width) refuse("logits must have a row for each of the scores");
    if (vocab < 1 || vocab > 1 << 20) refuse("a vocabulary of 1 to 2^20 tokens");
    if (rows > INT32_MAX) refuse("too many rows for one call");
    if (k > width * vocab) refuse("%lld candidates of %lld there are", (long long)k, (long long)(width * vocab));
    if (eos >= 0 && k < beams + width)
      refuse("with eos, %lld beams after %lld need at least %lld candidates", (long long)beams, (long long)width, (long long)(beams + width));
    if (logits.stride(1) != 1 || (rows > 1 && logits.stride(0) < vocab)) logits = logits.clone(at::MemoryFormat::Contiguous);
    rtr_beam_step s = {};
    at::Tensor allowed;
    if (a[7] != Py_None) {
      allowed = tensor(a[7], "allowed");
      if (allowed.scalar_type() != at::kBool || !here(allowed, index) || allowed.dim() < 1 || allowed.dim() > 2 ||
          allowed.size(-1) != vocab || (allowed.dim() == 2 && allowed.size(0) != rows && allowed.size(0) != 1))
        refuse("allowed must be bool [items * beams, vocab] or [vocab] on the handle's device");
      const bool one = allowed.dim() == 1 || allowed.size(0) == 1 || allowed.stride(0) == 0;
      if ((vocab > 1 && allowed.stride(-1) != 1) || (!one && allowed.stride(0) < vocab))
        allowed = allowed.clone(at::MemoryFormat::Contiguous);
      s.allowed = static_cast<const uint8_t*>(allowed.data_ptr());
      s.allowed_stride = allowed.dim() == 1 || allowed.size(0) == 1 ? 0 : allowed.stride(0);
    }
    if (items > INT32_MAX / 256) refuse("too many items for one call");
    Room out(index, 3 * (Room::of(items * k, 4) + Room::of(items * beams, 4)));
    const at::Tensor all_tokens = out.take({items, k}, at::kInt), all_parents = out.take({items, k}, at::kInt),
                     all_scores = out.take({items, k}, at::kFloat), tokens = out.take({items, beams}, at::kInt),
                     parents = out.take({items, beams}, at::kInt), next = out.take({items, beams}, at::kFloat);
    s.logits = logits.data_ptr();
    s.scores = static_cast<const float*>(scores.data_ptr());
    s.logits_stride = rows > 1 ? logits.stride(0) : vocab;
    s.dtype = type_of(logits);
    s.items = (int32_t)items;
    s.n = (int32_t)width;
    s.vocab = (int32_t)vocab;
    s.k = (int32_t)k;
    s.beams = (int32_t)beams;
    s.eos = eos > INT32_MAX ? -1 : (int32_t)eos;
    s.all_tokens = static_cast<int32_t*>(all_tokens.data_ptr());
    s.all_parents = static_cast<int32_t*>(all_parents.data_ptr());
    s.all_scores = static_cast<float*>(all_scores.data_ptr());
    s.next_tokens = static_cast<int32_t*>(tokens.data_ptr());
    s.next_parents = static_cast<int32_t*>(parents.data_ptr());
    s.next_scores = static_cast<float*>(next.data_ptr());
    s.status = status;
    int64_t room = 0;
    check(beam_workspace(&s, index, &room));
    at::Tensor work = room_for(index, {room}, at::kByte);
    check(beam_select(&s, work.data_ptr(), room, index, stream_of(index)));
    return tuple_of({tokens, parents, next, all_tokens, all_parents, all_scores});
  });
}

// A state's layout: its dimensions but that of the rows, outermost first, as few as its strides allow; false where
// it holds nothing.
bool layout_of(const at::Tensor& t, int64_t dim, int64_t token_dim, int64_t tokens, rtr_beam_state& s) {
  struct Dim { int64_t size, stride; };
  Dim dims[16];
  int n = 0;
  const int64_t size = t.element_size();
  for (int64_t d = 0; d < t.dim(); ++d) {
    const int64_t count = d == token_dim ? tokens : t.size(d);
    if (!count) return false;
    if (d == dim || count == 1) continue;
    if (n == 16) refuse("a state has too many dimensions");
    dims[n++] = Dim{count, t.stride(d)};
  }
  std::sort(dims, dims + n, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  Dim with_rows[17];
  std::copy(dims, dims + n, with_rows);
  int all = n;
  if (t.size(dim) > 1) with_rows[all++] = Dim{t.size(dim), t.stride(dim)};
  std::sort(with_rows, with_rows + all, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  int64_t reach = 0;
  for (int i = all - 1; i >= 0; --i) {
    if (with_rows[i].stride <= reach) refuse("the values of a state overlap in memory");
    reach += (with_rows[i].size - 1) * with_rows[i].stride;
  }
  s = {};
  s.data = t.data_ptr();
  s.row_bytes = (t.size(dim) > 1 ? t.stride(dim) : 1) * size;
  s.inner = size;
  while (n && dims[n - 1].stride * size == s.inner) s.inner *= dims[--n].size;
  int out = 0;
  Dim outer[16];
  for (int i = 0; i < n; ++i) {
    if (out && outer[out - 1].stride == dims[i].stride * dims[i].size) outer[out - 1] = Dim{outer[out - 1].size * dims[i].size, dims[i].stride};
    else outer[out++] = dims[i];
  }
  if (out > 3) refuse("a state's rows lie in more than three strided dimensions: reorder a contiguous one");
  for (int d = 0; d < 3; ++d) s.sizes[d] = 1;
  for (int i = 0; i < out; ++i) {
    if (outer[i].size > INT32_MAX) refuse("a state's dimensions must fit 32 bits");
    s.sizes[3 - out + i] = (int32_t)outer[i].size;
    s.strides[3 - out + i] = outer[i].stride * size;
  }
  return true;
}

// reorder(status address, device, beams, states (a tensor, list or tuple), parents, dim, token_dim or None, tokens or None)
PyObject* call_reorder(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    uint32_t* status = static_cast<uint32_t*>(PyLong_AsVoidPtr(a[0]));
    const int index = (int)PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) throw Raised{};
    const int64_t beams = whole(a[2], "beams"), dim_ = whole(a[5], "dim");
    const at::Tensor& parents = tensor(a[4], "parents");
    if (parents.scalar_type() != at::kInt || parents.dim() != 2 || parents.size(1) != beams || !parents.is_contiguous() ||
        !here(parents, index))
      refuse("parents must be int32 [items, %lld], contiguous, on the handle's device", (long long)beams);
    const int64_t items = parents.size(0);
    if (items > 65535) refuse("at most 65535 items in one call");
    if ((a[6] == Py_None) != (a[7] == Py_None)) refuse("token_dim and tokens belong together");
    const bool one = THPVariable_Check(a[3]);
    if (!one && !PyList_Check(a[3]) && !PyTuple_Check(a[3])) refuse("states must be a tensor, or a list or tuple of them");
    const Py_ssize_t count = one ? 1 : PySequence_Fast_GET_SIZE(a[3]);
    std::vector<rtr_beam_state> states;
    std::vector<const void*> known;
    states.reserve(count);
    known.reserve(count);
    for (int pass = 0; pass < 2; ++pass) {  // all are looked at before any counts as written
      for (Py_ssize_t i = 0; i < count; ++i) {
        const at::Tensor& t = tensor(one ? a[3] : PySequence_Fast_GET_ITEM(a[3], i), "a state");
        if (pass) {
          written(t, "a state");
          continue;
        }
        if (t.requires_grad()) refuse("a state must not require a gradient");
        const int64_t rank = t.dim(), dim = dim_ < 0 ? dim_ + rank : dim_;
        if (!here(t, index) || dim < 0 || dim >= rank || t.size(dim) != items * beams)
          refuse("dimension dim of a state must be the %lld rows, on the handle's device", (long long)(items * beams));
        if (t.is_complex() || t.is_quantized() || t.layout() != at::kStrided) refuse("a state must be a plain tensor");
        int64_t token_dim = -1, tokens = 0;
        if (a[6] != Py_None) {
          token_dim = whole(a[6], "token_dim");
          tokens = whole(a[7], "tokens");
          if (token_dim < 0) token_dim += rank;
          if (token_dim < 0 || token_dim >= rank || token_dim == dim) refuse("token_dim must be another dimension than dim");
          if (tokens < 0 || tokens > t.size(token_dim)) refuse("a state holds %lld tokens", (long long)t.size(token_dim));
        }
        rtr_beam_state s;
        if (layout_of(t, dim, token_dim, tokens, s)) {
          states.push_back(s);
          known.push_back(s.data);
        }
      }
      if (!pass) {
        std::sort(known.begin(), known.end());
        if (std::adjacent_find(known.begin(), known.end()) != known.end()) refuse("a state is among the states twice");
      }
    }
    check(beam_reorder(states.data(), (int32_t)states.size(), static_cast<const int32_t*>(parents.data_ptr()), (int32_t)items,
                       (int32_t)beams, status, index, stream_of(index)));
    Py_RETURN_NONE;
  });
}

// setup(addresses of the entry points in the order below, last_error's, NativeError)
PyObject* call_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    void* at[7];
    for (int i = 0; i < 7; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) throw Raised{};
    pages_grow = reinterpret_cast<decltype(pages_grow)>(at[0]);
    pages_release = reinterpret_cast<decltype(pages_release)>(at[1]);
    rotary = reinterpret_cast<decltype(rotary)>(at[2]);
    beam_workspace = reinterpret_cast<decltype(beam_workspace)>(at[3]);
    beam_select = reinterpret_cast<decltype(beam_select)>(at[4]);
    beam_reorder = reinterpret_cast<decltype(beam_reorder)>(at[5]);
    last_error = reinterpret_cast<decltype(last_error)>(at[6]);
    Py_INCREF(a[7]);
    Py_XSETREF(native_error, a[7]);
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {{"setup", CALL(call_setup)},
                         {"grow", CALL(call_grow)},
                         {"release", CALL(call_release)},
                         {"rotate", CALL(call_rotate)},
                         {"select", CALL(call_select)},
                         {"reorder", CALL(call_reorder)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_op_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__op_call() { return PyModule_Create(&module); }
