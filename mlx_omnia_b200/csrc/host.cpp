// The host's side of the calls of a step of drafted tokens and of logits' options: checks of arguments, memory for what is made, the
// arguments' record and the launch, in one call from Python. (Small steps are bound by the host: the same in Python took 12 to 24 us a call.)
// Compiled with the host's compiler against the torch that is installed; the kernels' launchers are called by address. Records are laid out as in
// drafted.cu, attention_tree.cuh and logits.cu.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <string>
#include <vector>

namespace {

constexpr int64_t MOST_DRAFTED = 256, MOST_GROUPS = 8, MOST_KINDS = 8;

PyObject* kernel_error = nullptr;   // ops.KernelError
PyObject* memory_error = nullptr;   // torch.OutOfMemoryError
PyObject* error_address = nullptr;  // device index -> address of the word that kernels report in
int64_t error_addresses[64] = {};

struct Refused {
  std::string why;
};
struct Raised {};  // a Python error is set

[[noreturn]] void refuse(const char* what, const std::string& why) { throw Refused{std::string(what) + why}; }

std::string shape_text(at::IntArrayRef shape) {
  std::string text = "[";
  for (size_t i = 0; i < shape.size(); ++i) text += (i ? ", " : "") + std::to_string(shape[i]);
  return text + "]";
}

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) refuse(what, std::string(": ") + name + " is a tensor, not a " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t index_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

[[noreturn]] void wrong(const char* what, const char* name, const at::Tensor& t, at::ScalarType type, int64_t index, const std::string& shape) {
  if (index_of(t) != index) refuse(what, std::string(": ") + name + " lies on " + t.device().str() + ", not with the other tensors");
  refuse(what, std::string(": ") + name + " is a contiguous " + c10::toString(type) + " tensor of " + shape + ", not " + c10::toString(t.scalar_type()) + " " +
                   shape_text(t.sizes()) + " with strides " + shape_text(t.strides()));
}
// A contiguous tensor of this type and shape on device `index`. -> its address
void* like(PyObject* o, const char* what, const char* name, at::ScalarType type, int64_t index, std::initializer_list<int64_t> shape) {
  const at::Tensor& t = tensor(o, what, name);
  if (t.scalar_type() != type || !t.sizes().equals(at::IntArrayRef(shape.begin(), shape.size())) || !t.is_contiguous() || index_of(t) != index)
    wrong(what, name, t, type, index, shape_text(at::IntArrayRef(shape.begin(), shape.size())));
  return t.data_ptr();
}
// The size of a contiguous tensor of one dimension.
int64_t list_of(PyObject* o, const char* what, const char* name, at::ScalarType type, int64_t index) {
  const at::Tensor& t = tensor(o, what, name);
  if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || index_of(t) != index) wrong(what, name, t, type, index, "[n]");
  return t.size(0);
}
int64_t whole(PyObject* o, const char* what, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(": ") + name + " is a whole number");
  }
  return v;
}
// So many positions, or (beyond 31 bits) more than a request holds.
int positions(PyObject* o, const char* what, const char* name) {
  const int64_t v = whole(o, what, name);
  if (v < 0) refuse(what, std::string(": ") + name + " is no negative number");
  return (int)(v < (1LL << 31) - MOST_DRAFTED ? v : (1LL << 31) - MOST_DRAFTED);
}
int64_t address(PyObject* o) { return (int64_t)PyLong_AsLongLong(o); }
double real(PyObject* o, const char* what, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(": ") + name + " is a number");
  }
  return v;
}
PyObject* item(PyObject* tuple, Py_ssize_t i, Py_ssize_t of, const char* what) {
  if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != of) refuse(what, std::string(" takes a tuple of ") + std::to_string(of));
  return PyTuple_GET_ITEM(tuple, i);
}

// The current stream of device `index`, which has to be the current one (a launch goes to its stream).
void* stream_of(const char* what, int64_t index) {
  if (index < 0) refuse(what, " takes tensors on a CUDA device");
  if (c10::cuda::current_device() != index)
    refuse(what, " takes tensors on the current CUDA device (" + std::to_string((int)c10::cuda::current_device()) + "), not on " + std::to_string(index));
  return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
}
void* error_word(int64_t index) {
  if (index >= 64) refuse("a device", " beyond the 64th");
  if (!error_addresses[index]) {
    PyObject* found = PyObject_CallFunction(error_address, "L", (long long)index);
    if (!found) throw Raised{};
    error_addresses[index] = address(found);
    Py_DECREF(found);
  }
  return (void*)error_addresses[index];
}
void check(int code, const char* what) {
  if (code != 0) refuse(what, ": CUDA error " + std::to_string(code) + " at launch (bad sizes for this kernel, or an earlier fault)");
}

at::Tensor empty(int64_t index, at::ScalarType type, at::IntArrayRef shape) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, (c10::DeviceIndex)index)));
}
// Part of a buffer of 4-byte numbers as a tensor of its own, from number `at` on.
at::Tensor part_of(const at::Tensor& buffer, int64_t at, at::ScalarType type, at::IntArrayRef shape) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buffer.storage()), buffer.key_set(), c10::scalarTypeToTypeMeta(type));
  c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  impl->set_storage_offset(at * 4 / (int64_t)c10::elementSize(type));
  impl->set_sizes_contiguous(shape);
  return t;
}
PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(kernel_error, r.why.c_str());
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(memory_error, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
void count(const char* what, Py_ssize_t given, Py_ssize_t wanted) {
  if (given != wanted) refuse(what, ": " + std::to_string(given) + " arguments in place of " + std::to_string(wanted));
}

// ---- step_tables ---------------------------------------------------------------------------------------------------------------------
struct TableGroup {
  const void *pages, *starts;
  void *table, *slots;
  long long count;
  int width, stride;
};
struct Tables {
  const void *held, *brought, *parents;
  void *positions, *cu_seqlens, *seq_lens, *ancestors, *err;
  int requests, tokens, page_size, words, groups, unused;
  TableGroup group[MOST_GROUPS];
};
static_assert(sizeof(TableGroup) == 48 && sizeof(Tables) == 88 + 48 * MOST_GROUPS, "as in drafted.cu");

// (entry, held, brought, lists, page_size, tokens, parents, most) -> (positions, cu_seqlens, seq_lens, [(table, slots)], ancestors)
PyObject* step_tables(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    const char* what = "step_tables";
    count(what, given, 8);
    const at::Tensor& held = tensor(args[1], what, "held");
    const int64_t index = index_of(held), n = list_of(args[1], what, "held", at::kInt, index), page_size = whole(args[4], what, "page_size"),
                  tokens = whole(args[5], what, "tokens");
    Tables a = {};
    a.held = held.data_ptr(), a.brought = like(args[2], what, "brought", at::kInt, index, {n});
    int64_t words = 0;
    if (args[7] != Py_None) {
      const int64_t most = whole(args[7], what, "most");
      if (most < 1 || most > MOST_DRAFTED)
        refuse(what, ": a request brings 1 to " + std::to_string(MOST_DRAFTED) + " drafted tokens, not " + std::to_string(most));
      words = (most + 31) / 32;
    }
    if (args[6] != Py_None) {
      if (!words) refuse(what, ": parents go with `most`, the most tokens that a request brings");
      a.parents = like(args[6], what, "parents", at::kInt, index, {tokens});
    }
    PyObject* lists = PySequence_Fast(args[3], "step_tables takes a list of PageLists");
    if (!lists) throw Raised{};
    struct Release {
      PyObject* o;
      ~Release() { Py_DECREF(o); }
    } release{lists};
    const int64_t groups = PySequence_Fast_GET_SIZE(lists);
    if (n < 1 || n > 65534 || tokens < 0 || tokens >= (1LL << 31) || page_size < 1 || page_size >= (1LL << 31) || groups > MOST_GROUPS)
      refuse(what, " takes 1 to 65,534 requests, pages of a token or more and up to " + std::to_string(MOST_GROUPS) + " groups");
    int64_t size = 2 * tokens * groups;  // one buffer: the slots (8 bytes each) first, then all that has 4
    for (int64_t g = 0; g < groups; ++g) {
      PyObject* x = PySequence_Fast_GET_ITEM(lists, g);
      PyObject *pages = item(x, 0, 4, what), *starts = item(x, 1, 4, what);
      TableGroup& group = a.group[g];
      group.count = list_of(pages, what, "pages", at::kInt, index);
      group.pages = THPVariable_Unpack(pages).data_ptr(), group.starts = like(starts, what, "starts", at::kLong, index, {n});
      const int64_t width = whole(item(x, 2, 4, what), what, "width"), stride = whole(item(x, 3, 4, what), what, "stride");
      if (width < 1 || stride < 1 || width >= (1LL << 31) || stride >= (1LL << 31) || (stride > 1 && words))
        refuse(what, ": tables have a column or more, and drafted tokens a stored row each");
      group.width = (int)width, group.stride = (int)stride;
      size += n * width;
    }
    void* stream = stream_of(what, index);
    a.err = error_word(index);
    const at::Tensor buffer = empty(index, at::kInt, {size + tokens + 2 * n + 1 + tokens * words});
    int* base = buffer.data_ptr<int>();
    int64_t at = 2 * tokens * groups;
    PyObject* tables = PyList_New(groups);
    for (int64_t g = 0; g < groups; ++g) {
      TableGroup& group = a.group[g];
      group.slots = base + 2 * tokens * g, group.table = base + at;
      PyObject* pair = PyTuple_New(2);
      PyTuple_SET_ITEM(pair, 0, wrap(part_of(buffer, at, at::kInt, {n, (int64_t)group.width})));
      PyTuple_SET_ITEM(pair, 1, wrap(part_of(buffer, 2 * tokens * g, at::kLong, {tokens})));
      PyList_SET_ITEM(tables, g, pair);
      at += n * group.width;
    }
    const int64_t positions = at, cu = positions + tokens, lens = cu + n + 1, sees = lens + n;
    a.positions = base + positions, a.cu_seqlens = base + cu, a.seq_lens = base + lens, a.ancestors = words ? base + sees : nullptr;
    a.requests = (int)n, a.tokens = (int)tokens, a.page_size = (int)page_size, a.words = (int)words, a.groups = (int)groups;
    const int code = ((int (*)(const void*, void*))address(args[0]))(&a, stream);
    if (code) Py_DECREF(tables);
    check(code, what);
    PyObject* made = PyTuple_New(5);
    PyTuple_SET_ITEM(made, 0, wrap(part_of(buffer, positions, at::kInt, {tokens})));
    PyTuple_SET_ITEM(made, 1, wrap(part_of(buffer, cu, at::kInt, {n + 1})));
    PyTuple_SET_ITEM(made, 2, wrap(part_of(buffer, lens, at::kInt, {n})));
    PyTuple_SET_ITEM(made, 3, tables);
    if (words) PyTuple_SET_ITEM(made, 4, wrap(part_of(buffer, sees, at::kInt, {tokens, words})));
    else PyTuple_SET_ITEM(made, 4, Py_NewRef(Py_None));
    return made;
  });
}

// ---- accept_drafts, keep_rows --------------------------------------------------------------------------------------------------------
// (entry, chosen, token_ids, ancestors, cu_seqlens) -> (path, kept, tokens)
PyObject* accept_drafts(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    const char* what = "accept_drafts";
    count(what, given, 5);
    const at::Tensor& ancestors = tensor(args[3], what, "ancestors");
    const int64_t index = index_of(ancestors), tokens = ancestors.dim() == 2 ? ancestors.size(0) : 0, words = ancestors.dim() == 2 ? ancestors.size(1) : 0;
    const int64_t n = list_of(args[4], what, "cu_seqlens", at::kInt, index) - 1;
    if (n < 1 || n >= (1LL << 31) || words < 1 || words > MOST_DRAFTED / 32)
      refuse(what, " takes a request or more, of " + std::to_string(MOST_DRAFTED) + " tokens at most");
    const void* sees = like(args[3], what, "ancestors", at::kInt, index, {tokens, words});
    const void* chosen = like(args[1], what, "chosen", at::kInt, index, {tokens});
    const void* ids = like(args[2], what, "token_ids", at::kInt, index, {tokens});
    void* stream = stream_of(what, index);
    const at::Tensor buffer = empty(index, at::kInt, {n * (32 * words + 2)});
    int* base = buffer.data_ptr<int>();
    const int64_t kept = n * 32 * words, last = kept + n;
    using Entry = int (*)(const void*, const void*, const void*, const void*, int, int, void*, void*, void*, int, void*, void*);
    check(((Entry)address(args[0]))(chosen, ids, sees, THPVariable_Unpack(args[4]).data_ptr(), (int)n, (int)words, base, base + kept, base + last, (int)tokens,
                                    error_word(index), stream),
          what);
    PyObject* made = PyTuple_New(3);
    PyTuple_SET_ITEM(made, 0, wrap(part_of(buffer, 0, at::kInt, {n, 32 * words})));
    PyTuple_SET_ITEM(made, 1, wrap(part_of(buffer, kept, at::kInt, {n})));
    PyTuple_SET_ITEM(made, 2, wrap(part_of(buffer, last, at::kInt, {n})));
    return made;
  });
}

// (entry, pages, rows, page_size, block_table, held, path, kept)
PyObject* keep_rows(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    const char* what = "keep_rows";
    count(what, given, 8);
    const at::Tensor &pages = tensor(args[1], what, "pages"), &table = tensor(args[4], what, "block_table"), &path = tensor(args[6], what, "path");
    if (table.dim() != 2 || path.dim() != 2 || pages.dim() < 3)
      refuse(what, " takes pages [layers, pages, ...], a block table [requests, pages] and paths [requests, tokens]");
    const int64_t index = index_of(pages), n = table.size(0), width = table.size(1), most = path.size(1), page_size = whole(args[3], what, "page_size");
    like(args[4], what, "block_table", at::kInt, index, {n, width});
    const void* held = like(args[5], what, "held", at::kInt, index, {n});
    like(args[6], what, "path", at::kInt, index, {n, most});
    const void* kept = like(args[7], what, "kept", at::kInt, index, {n});
    if (!pages.is_contiguous()) refuse(what, " takes contiguous pages");
    int64_t elements = 1, sum = 0, item_size = (int64_t)pages.element_size();
    for (int64_t i = 2; i < pages.dim(); ++i) elements *= pages.size(i);
    PyObject* rows = args[2];
    const Py_ssize_t kinds = PyTuple_Check(rows) ? PyTuple_GET_SIZE(rows) : 0;
    int heads[MOST_KINDS], bytes[MOST_KINDS];
    bool good = kinds >= 1 && kinds <= MOST_KINDS && page_size >= 1;
    for (Py_ssize_t k = 0; k < kinds && good; ++k) {
      const int64_t h = whole(item(PyTuple_GET_ITEM(rows, k), 0, 2, what), what, "heads"), w = whole(item(PyTuple_GET_ITEM(rows, k), 1, 2, what), what, "width");
      good = h >= 1 && w >= 1 && h < (1 << 24) && w < (1 << 24);
      heads[k] = (int)h, bytes[k] = (int)(w * item_size), sum += h * w;
    }
    if (!good || sum * page_size != elements)
      refuse(what, ": pages of " + std::to_string(elements) + " elements do not hold " + std::to_string(page_size) + " such rows");
    if (most < 1 || most > MOST_DRAFTED || n < 1 || n >= (1LL << 31) || width < 1 || pages.size(0) < 1 || pages.size(0) > 65535 || pages.size(1) < 1 ||
        pages.size(1) >= (1LL << 31))
      refuse(what, " takes a request or more, with paths of 1 to " + std::to_string(MOST_DRAFTED) + " tokens, and pages of a layer or more");
    void* stream = stream_of(what, index);
    using Entry = int (*)(void*, long long, long long, int, int, int, const int*, const int*, int, const void*, int, const void*, const void*, const void*, int, int,
                          void*, void*);
    check(((Entry)address(args[0]))(pages.data_ptr(), pages.size(1) * elements * item_size, elements * item_size, (int)pages.size(0), (int)pages.size(1),
                                    (int)page_size, heads, bytes, (int)kinds, table.data_ptr(), (int)width, held, path.data_ptr(), kept, (int)n, (int)most,
                                    error_word(index), stream),
          what);
    Py_RETURN_NONE;
  });
}

// ---- tree_attention ------------------------------------------------------------------------------------------------------------------
struct Tree {
  const void *q, *k_pages, *v_pages, *gate;
  void* out;
  const void *block_table, *cu_seqlens, *seq_lens, *positions, *ancestors, *sink;
  void *part_o, *part_ml, *err, *items;
  long long page_stride;
  int tokens, requests, max_pages, num_pages, nq, nkv, d, dv, page_size, gate_stride, words, window, keep, run, chunk, parts;
  float scale, softcap;
};
static_assert(sizeof(Tree) == 200, "as in attention_tree.cuh");

// (entry, merge, kind, q, pages, block_table, cu_seqlens, seq_lens, positions, ancestors, gate, gate_col, sink, nkv, dk, dv, page_size, requests, most,
// window, keep, run, chunk, parts, slots, tile, scale, softcap) -> out. `kind`: what follows the record in the entry's arguments: 0 most, parts; 1
// most, tile, parts; 2 most, dtype, and where there are several parts the merge. `slots`: rows of partial sums.
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    const char* what = "tree_attention";
    count(what, given, 28);
    const at::Tensor &q = tensor(args[3], what, "q"), &pages = tensor(args[4], what, "pages"), &table = tensor(args[5], what, "block_table"),
                     &ancestors = tensor(args[9], what, "ancestors");
    if (q.dim() != 3 || !q.is_contiguous()) refuse(what, " takes contiguous queries [tokens, heads, width]");
    const int64_t index = index_of(q), tokens = q.size(0), nq = q.size(1), d = q.size(2), nkv = whole(args[13], what, "nkv"), dk = whole(args[14], what, "dk"),
                  dv = whole(args[15], what, "dv"), page_size = whole(args[16], what, "page_size"), n = whole(args[17], what, "requests"),
                  most = whole(args[18], what, "most"), gate_col = whole(args[11], what, "gate_col");
    const at::ScalarType type = q.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse("kernels", std::string(" take float32 or bfloat16, not ") + c10::toString(type));
    const int64_t size = (int64_t)q.element_size();
    if (dk != d || nkv < 1 || nq % nkv || pages.scalar_type() != type || d < 1 || d > 512 || dv < 1 || dv > 512 || !pages.is_contiguous() || index_of(pages) != index ||
        pages.dim() < 2 || pages.size(0) * nkv * (dk + dv) * page_size != pages.numel())
      refuse(what, ": " + std::to_string(nq) + " heads of " + std::to_string(d) + " (" + c10::toString(type) + ") do not go with a cache of " + std::to_string(nkv) +
                       " heads of " + std::to_string(dk) + " and " + std::to_string(dv) + " (" + c10::toString(pages.scalar_type()) + ", " + pages.device().str() + ")");
    if (table.dim() != 2 || ancestors.dim() != 2) refuse(what, " takes a block table [requests, pages] and ancestors [tokens, words]");
    const int64_t width = table.size(1), words = ancestors.size(1);
    Tree a = {};
    a.ancestors = like(args[9], what, "ancestors", at::kInt, index, {tokens, words});
    a.positions = like(args[8], what, "positions", at::kInt, index, {tokens});
    a.block_table = like(args[5], what, "block_table", at::kInt, index, {n, width});
    a.cu_seqlens = like(args[6], what, "cu_seqlens", at::kInt, index, {n + 1});
    a.seq_lens = like(args[7], what, "seq_lens", at::kInt, index, {n});
    if (most < 1 || most > 32 * words || 32 * words > MOST_DRAFTED || n < 1 || width < 1 || tokens >= (1LL << 31))
      refuse(what, ": a request brings up to " + std::to_string(most) + " tokens, the tree has " + std::to_string(words) + " words for each (" +
                       std::to_string(MOST_DRAFTED) + " tokens at most)");
    if (args[10] != Py_None) {
      const at::Tensor& gate = tensor(args[10], what, "gate");
      if (gate.scalar_type() != type || gate.dim() != 2 || gate.stride(1) != 1 || gate.size(0) != tokens || index_of(gate) != index || gate_col < 0 ||
          gate_col > gate.size(1) - nq * dv || (tokens > 1 && gate.stride(0) < gate.size(1)))
        refuse(what, ": the gate's " + std::to_string(nq * dv) + " columns from " + std::to_string(gate_col) + " on lie outside rows of " + shape_text(gate.sizes()) +
                         ", or are of another type");
      a.gate = (const char*)gate.data_ptr() + gate_col * size, a.gate_stride = (int)gate.stride(0);
    }
    if (args[12] != Py_None) a.sink = like(args[12], what, "sink", at::kFloat, index, {nq});
    void* stream = stream_of(what, index);
    at::Tensor out = empty(index, type, {tokens, nq * dv});
    if (tokens == 0) return wrap(std::move(out));
    const int64_t slots = whole(args[24], what, "slots"), kind = whole(args[2], what, "kind"), parts = whole(args[23], what, "parts");
    at::Tensor part;
    if (slots) {
      // Rows of sums, then their offsets and sums of weights, which are read in pairs: on a multiple of 16 bytes whatever the widths. Of the kernels by
      // equal shares where the join finds each tile of rows, ahead of both.
      const int64_t tile = whole(args[25], what, "tile"), ahead = kind < 2 ? 4 * n * nkv * ((most * (nq / nkv) + tile - 1) / tile) : 0;
      const int64_t sums = (slots * dv + 3) / 4 * 4;
      part = empty(index, at::kFloat, {ahead + sums + 2 * slots});
      a.items = part.data_ptr(), a.part_o = part.data_ptr<float>() + ahead, a.part_ml = part.data_ptr<float>() + ahead + sums;
    }
    a.q = q.data_ptr(), a.k_pages = pages.data_ptr(), a.v_pages = (const char*)a.k_pages + nkv * dk * page_size * size, a.out = out.data_ptr();
    a.err = error_word(index), a.page_stride = nkv * (dk + dv) * page_size;
    a.tokens = (int)tokens, a.requests = (int)n, a.max_pages = (int)width, a.num_pages = (int)pages.size(0), a.nq = (int)nq, a.nkv = (int)nkv, a.d = (int)d;
    a.dv = (int)dv, a.page_size = (int)page_size, a.words = (int)words, a.window = positions(args[19], what, "window"), a.keep = positions(args[20], what, "keep_first");
    a.run = positions(args[21], what, "chunk"), a.chunk = (int)whole(args[22], what, "plan"), a.parts = (int)parts;
    a.scale = (float)real(args[26], what, "scale"), a.softcap = (float)real(args[27], what, "softcap");
    const int64_t entry = address(args[0]);
    const int dtype = type == at::kBFloat16;
    if (kind == 0) {
      check(((int (*)(const void*, int, int, void*))entry)(&a, (int)most, (int)parts, stream), what);
    } else if (kind == 1) {
      check(((int (*)(const void*, int, int, int, void*))entry)(&a, (int)most, (int)whole(args[25], what, "tile"), (int)parts, stream), what);
    } else {
      check(((int (*)(const void*, int, int, void*))entry)(&a, (int)most, dtype, stream), what);
      if (parts > 1) check(((int (*)(const void*, int, void*))address(args[1]))(&a, dtype, stream), what);
    }
    return wrap(std::move(out));
  });
}

// ---- adjust_logits -------------------------------------------------------------------------------------------------------------------
struct Adjust {
  const void* logits;
  void* out;
  const void *requests, *history, *starts, *lengths, *prompts, *contexts, *repetition, *frequency, *presence, *bias_ids, *bias_values, *bias_starts, *mask_words,
      *mask_rows, *ancestors, *token_ids, *cu_seqlens, *nodes;
  void* err;
  long long stride, out_stride, history_tokens, bias_count;
  int rows, vocab, num_requests, masks, mask_width, words, tokens, unused, penalised, padding;
};
static_assert(sizeof(Adjust) == 240, "as in logits.cu");

// (entry, logits, history, repetition, frequency, presence, contexts, requests, bias, masks, drafted, out) -> the tensor written
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    const char* what = "adjust_logits";
    count(what, given, 12);
    const at::Tensor& logits = tensor(args[1], what, "logits");
    if (logits.dim() != 2 || logits.scalar_type() != at::kFloat || logits.stride(1) != 1)
      refuse(what, " takes float32 logits [rows, vocab] whose rows lie in one piece");
    const int64_t index = index_of(logits), rows = logits.size(0), vocab = logits.size(1), stride = logits.stride(0);
    if (rows > 1 && stride < vocab) refuse(what, " takes rows that lie apart");
    if (rows > 65535 || vocab >= (1LL << 30)) refuse(what, " takes up to 65,535 rows of fewer than 2^30 logits");
    PyObject *history = args[2], *bias = args[8], *masks = args[9], *drafted = args[10];
    Adjust a = {};
    int64_t num = rows;
    const bool text = history != Py_None, biased = bias != Py_None;
    if (text) {
      PyObject* tokens = item(history, 0, 4, what);
      num = list_of(item(history, 2, 4, what), what, "lengths", at::kInt, index);
      a.history_tokens = list_of(tokens, what, "tokens", at::kInt, index);
      a.history = THPVariable_Unpack(tokens).data_ptr();
      a.starts = like(item(history, 1, 4, what), what, "starts", at::kLong, index, {num});
      a.lengths = THPVariable_Unpack(item(history, 2, 4, what)).data_ptr();
      a.prompts = like(item(history, 3, 4, what), what, "prompts", at::kInt, index, {num});
    }
    const void** penalties[3] = {&a.repetition, &a.frequency, &a.presence};
    static const char* names[3] = {"repetition", "frequency", "presence"};
    for (int i = 0; i < 3; ++i)
      if (args[3 + i] != Py_None) {
        if (!text) refuse(what, ": penalties go by the requests' history");
        *penalties[i] = like(args[3 + i], what, names[i], at::kFloat, index, {num});
        a.penalised = 1;
      }
    if (args[6] != Py_None) {
      if (!text) refuse(what, ": penalties go by the requests' history");
      a.contexts = like(args[6], what, "contexts", at::kInt, index, {num});
    }
    if (biased) {
      PyObject *ids = item(bias, 0, 3, what), *starts = item(bias, 2, 3, what);
      a.bias_count = list_of(ids, what, "ids", at::kInt, index);
      if (!text) num = list_of(starts, what, "bias starts", at::kInt, index) - 1;
      if (num < 0) refuse(what, ": bias starts are one more than the requests");
      a.bias_starts = like(starts, what, "bias starts", at::kInt, index, {num + 1});
      a.bias_values = like(item(bias, 1, 3, what), what, "values", at::kFloat, index, {(int64_t)a.bias_count});
      a.bias_ids = THPVariable_Unpack(ids).data_ptr();
    }
    if (args[7] != Py_None) {
      const void* requests = like(args[7], what, "requests", at::kInt, index, {rows});
      if (text || biased) a.requests = requests;  // (nothing else goes by them, and there is no number of requests then)
    } else if (num < rows && (text || biased)) {
      refuse(what, ": " + std::to_string(rows) + " rows of " + std::to_string(num) + " requests need `requests`");
    }
    if (masks != Py_None) {
      const at::Tensor& words = tensor(item(masks, 0, 2, what), what, "mask words");
      if (words.dim() != 2 || words.size(1) * 32 < vocab)
        refuse(what, ": masks are [masks, words] of " + std::to_string(vocab) + " tokens, 32 a word, not " + shape_text(words.sizes()));
      a.mask_words = like(item(masks, 0, 2, what), what, "mask words", at::kInt, index, {words.size(0), words.size(1)});
      a.mask_rows = like(item(masks, 1, 2, what), what, "mask rows", at::kInt, index, {rows});
      a.masks = (int)words.size(0), a.mask_width = (int)words.size(1);
    }
    if (drafted != Py_None) {
      PyObject* sees = item(item(drafted, 0, 4, what), 0, 1, what);
      const at::Tensor& ancestors = tensor(sees, what, "ancestors");
      if (ancestors.dim() != 2 || (text && args[7] == Py_None)) refuse(what, ": drafted rows need `requests`, and a tree of [tokens, words]");
      const int64_t tokens = ancestors.size(0), words = ancestors.size(1);
      const void* bits = like(sees, what, "ancestors", at::kInt, index, {tokens, words});
      const void* ids = like(item(drafted, 1, 4, what), what, "token_ids", at::kInt, index, {tokens});
      const int64_t of = list_of(item(drafted, 2, 4, what), what, "cu_seqlens", at::kInt, index);
      const void* nodes = like(item(drafted, 3, 4, what), what, "drafted rows", at::kInt, index, {rows});
      if (text && of != num + 1) refuse(what, ": drafted rows need the step of the same " + std::to_string(num) + " requests");
      if (a.penalised) {
        a.ancestors = bits, a.token_ids = ids, a.cu_seqlens = THPVariable_Unpack(item(drafted, 2, 4, what)).data_ptr(), a.nodes = nodes;
        a.tokens = (int)tokens, a.words = (int)words;
      }
    }
    at::Tensor out;
    bool same = false;
    if (args[11] == Py_None) {
      void* unused = stream_of(what, index);  // (ahead of the allocation: a tensor on the host is refused)
      (void)unused;
      out = empty(index, at::kFloat, {rows, vocab});
    } else {
      out = tensor(args[11], what, "out");
      if (out.scalar_type() != at::kFloat || !out.sizes().equals(logits.sizes()) || out.stride(1) != 1 || index_of(out) != index || (rows > 1 && out.stride(0) < vocab))
        refuse(what, " writes float32 rows that lie apart, in the logits' shape");
      const char *x = (const char*)logits.data_ptr(), *y = (const char*)out.data_ptr();
      same = x == y && (rows < 2 || out.stride(0) == stride);
      if (!same && rows && y < x + 4 * ((rows - 1) * stride + vocab) && x < y + 4 * ((rows - 1) * out.stride(0) + vocab))
        refuse(what, " writes to the logits themselves, or to a tensor that shares no memory with them");
    }
    void* stream = stream_of(what, index);
    if (rows && vocab) {
      a.logits = logits.data_ptr(), a.out = out.data_ptr(), a.err = error_word(index), a.stride = stride, a.out_stride = out.stride(0);
      a.rows = (int)rows, a.vocab = (int)vocab, a.num_requests = (int)num;
      check(((int (*)(const void*, int, void*))address(args[0]))(&a, same, stream), what);
    }
    return args[11] == Py_None ? wrap(std::move(out)) : Py_NewRef(args[11]);
  });
}

// (KernelError, torch.OutOfMemoryError, device index -> address of the error word)
PyObject* set_up(PyObject*, PyObject* const* args, Py_ssize_t given) {
  if (given != 3) {
    PyErr_SetString(PyExc_TypeError, "set_up takes two errors' classes and a function");
    return nullptr;
  }
  Py_XSETREF(kernel_error, Py_NewRef(args[0]));
  Py_XSETREF(memory_error, Py_NewRef(args[1]));
  Py_XSETREF(error_address, Py_NewRef(args[2]));
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(step_tables), METHOD(accept_drafts), METHOD(keep_rows), METHOD(tree_attention), METHOD(adjust_logits), METHOD(set_up), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "omnia_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_omnia_host() { return PyModule_Create(&module); }
