// What the Python calls do around the library's functions, one crossing from the interpreter to a call: outputs and
// zeroed words are made, addresses taken, the function called, results cut.  A call of a small bucket is bound by the
// host, and each of these steps costs a microsecond or two in the interpreter (an all-reduce of a 9 k-element bucket had
// some 65 us of it).
//
// A library function arrives as the ctypes object that stands for it, so that whoever replaces the library replaces it
// here too; ctypes lets other threads run while the function does.
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <limits>
#include <map>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "zen_hip.h"

namespace py = pybind11;
using at::Tensor;

namespace {

int64_t address(const Tensor &t) { return reinterpret_cast<int64_t>(t.data_ptr()); }

Tensor room(const Tensor &like, int64_t count, at::ScalarType type) {
  return at::empty({count}, like.options().dtype(type).requires_grad(false));
}

// What `make` returns, a call's new tensors, while other threads may hold the interpreter: an allocator that has to go to
// the device, or free memory first, takes its time (torch's own bindings let go of it too).
template <typename Make>
auto made(Make make) {
  py::gil_scoped_release others;
  return make();
}
using Two = std::tuple<Tensor, Tensor>;  // (in braces: made in this order)
using Three = std::tuple<Tensor, Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// Zeroed words for status words, counters and split sizes, cut from blocks that one fill zeroed.  Every piece is handed
// out once, in the order of the stream its block was made on.  One object to a host thread.
class Zeros {
 public:
  static constexpr int64_t kWords = 8192;
  static constexpr int64_t kSplit = 2;  // pieces begin at multiples of so many words: of 16 bytes, status words of 8

  Tensor words(const Tensor &like, int64_t stream, int64_t count) { return take(blocks_, like, stream, count, at::kLong, 0, nullptr); }
  Tensor status(const Tensor &like, int64_t stream) { return take(narrow_, like, stream, 1, at::kInt, 0, nullptr); }
  // `other`: a stream beside that uses the words too; *wait: it has to wait for the block's fill.
  Tensor words_for(const Tensor &like, int64_t stream, int64_t count, int64_t other, bool *wait) {
    return take(blocks_, like, stream, count, at::kLong, other, wait);
  }
  void fresh(int64_t device, int64_t stream) {
    blocks_.erase({device, stream});
    narrow_.erase({device, stream});
  }

 private:
  struct Block {
    Tensor all;
    int64_t used = 0;
    std::vector<int64_t> seen;
  };
  using Blocks = std::map<std::pair<int64_t, int64_t>, Block>;
  Blocks blocks_, narrow_;

  static Tensor take(Blocks &blocks, const Tensor &like, int64_t stream, int64_t count, at::ScalarType type, int64_t other,
                     bool *wait) {
    const auto options = like.options().dtype(type).requires_grad(false);
    if (count > kWords / 4) {
      if (wait) *wait = true;
      return at::zeros({count}, options);
    }
    Block &b = blocks[{like.device().index(), stream}];
    const int64_t step = (count + kSplit - 1) / kSplit * kSplit;
    if (!b.all.defined() || b.used + step > kWords) b = Block{at::zeros({kWords}, options), 0, {stream}};
    if (wait) {
      *wait = std::find(b.seen.begin(), b.seen.end(), other) == b.seen.end();
      if (*wait) b.seen.push_back(other);
    }
    const Tensor piece = b.all.narrow(0, b.used, count);
    b.used += step;
    return piece;
  }
};

// The covering view of one-dimensional tensors that sit back to back in one storage; none if they do not.
py::object one_buffer(const std::vector<Tensor> &tensors) {
  if (tensors.empty()) return py::none();
  const Tensor &first = tensors[0];
  if (first.dim() != 1 || !first.is_contiguous()) return py::none();
  const char *at = static_cast<const char *>(first.data_ptr());
  const void *storage = first.storage().data();
  const int64_t size = first.element_size();
  int64_t total = 0;
  for (const Tensor &t : tensors) {
    if (t.scalar_type() != first.scalar_type() || t.dim() != 1 || t.data_ptr() != at || !t.is_contiguous() ||
        t.storage().data() != storage)
      return py::none();
    total += t.numel();
    at += t.numel() * size;
  }
  return py::cast(first.as_strided({total}, {1}));
}

// Contiguous, of one type and on one device: what a kernel takes by their addresses.
bool plain_runs(const std::vector<Tensor> &tensors) {
  for (const Tensor &t : tensors)
    if (t.scalar_type() != tensors[0].scalar_type() || t.device() != tensors[0].device() || !t.is_contiguous()) return false;
  return true;
}

struct Lists {
  std::vector<int64_t> at, count;
  explicit Lists(const std::vector<Tensor> &tensors) {
    for (const Tensor &t : tensors) {
      at.push_back(address(t));
      count.push_back(t.numel());
    }
  }
  int64_t addresses() const { return reinterpret_cast<int64_t>(at.data()); }
  int64_t counts() const { return reinterpret_cast<int64_t>(count.data()); }
};

// Indices and values to their partitions.
py::tuple cut(const Tensor &indices, const Tensor &values, const std::vector<int64_t> &sizes) {
  int64_t total = 0;
  for (int64_t s : sizes) total += s;
  return py::make_tuple(at::split_with_sizes(indices.narrow(0, 0, total), sizes),
                        at::split_with_sizes(values.narrow(0, 0, total), sizes));
}

py::tuple load_balance(const py::object &fn, Zeros &zeros, const Tensor &flat, int code, int64_t m, int64_t partitions,
                       int rehash, const py::object &thr, int64_t k, const py::object &thr_out, int64_t capacity,
                       int64_t table, int64_t mode, const Tensor &ws, int64_t stream, int64_t host, int64_t words) {
  const auto [idx, val, splits, status] = made([&] {
    return Four{room(flat, capacity, at::kInt), room(flat, capacity, flat.scalar_type()), zeros.words(flat, stream, partitions),
                zeros.status(flat, stream)};
  });
  const py::object rc =
      host ? fn(address(flat), code, flat.numel(), m, partitions, rehash, thr, k, thr_out, address(idx), address(val),
                capacity, address(splits), table, mode, address(ws), ws.numel(), address(status), host, words, stream)
           : fn(address(flat), code, flat.numel(), m, partitions, rehash, thr, k, thr_out, address(idx), address(val),
                capacity, address(splits), table, mode, address(ws), ws.numel(), address(status), stream);
  return py::make_tuple(rc, idx, val, splits, status);
}

py::tuple merge(const py::object &fn, Zeros &zeros, const Tensor &indices, const Tensor &values, int code, int64_t dense_size,
                int64_t capacity, bool idx64, bool rounded, int64_t mode, const Tensor &ws, int64_t stream, int64_t host,
                int64_t words) {
  const auto [idx, val, count, status] = made([&] {
    return Four{room(values, capacity, idx64 ? at::kLong : at::kInt), room(values, capacity, rounded ? values.scalar_type() : at::kFloat),
                zeros.words(values, stream, 1), zeros.status(values, stream)};
  });
  const int from64 = indices.scalar_type() == at::kLong;
  const py::object rc =
      host ? fn(address(indices), from64, address(values), code, indices.numel(), dense_size, address(idx), idx64 ? 1 : 0,
                address(val), capacity, address(count), mode, address(ws), ws.numel(), address(status), host, words, stream)
           : fn(address(indices), from64, address(values), code, indices.numel(), dense_size, address(idx), idx64 ? 1 : 0,
                address(val), capacity, address(count), mode, address(ws), ws.numel(), address(status), stream);
  return py::make_tuple(rc, idx, val, count, status);
}

py::tuple select_count(const py::object &fn, Zeros &zeros, const Tensor &flat, int code, const py::object &thr, bool idx64,
                 int64_t capacity, const Tensor &ws, int64_t stream, int64_t host, int64_t words) {
  const auto [idx, val, count, status] = made([&] {
    return Four{room(flat, capacity, idx64 ? at::kLong : at::kInt), room(flat, capacity, flat.scalar_type()),
                zeros.words(flat, stream, 1), zeros.status(flat, stream)};
  });
  const py::object rc = fn(address(flat), code, flat.numel(), thr, address(idx), idx64 ? 1 : 0, address(val), capacity,
                           address(count), address(ws), ws.numel(), address(status), host, words, stream);
  return py::make_tuple(rc, idx, val);
}

py::tuple sample_threshold(const py::object &fn, Zeros &zeros, const Tensor &flat, int code, const Tensor &index, int64_t k,
                           const Tensor &ws, int64_t stream) {
  const auto [thr, status] = made([&] { return Two{room(flat, 2, at::kInt), zeros.status(flat, stream)}; });
  const py::object rc = fn(address(flat), code, flat.numel(), address(index), index.numel(), k, address(thr), address(ws),
                           ws.numel(), address(status), stream);
  return py::make_tuple(rc, thr, status);
}

py::tuple decode(const py::object &fn, Zeros &zeros, const Tensor &indices, const Tensor &values, int code, const Tensor &dense,
                 int64_t mode, const Tensor &ws, int64_t stream, int64_t host, int64_t words) {
  const Tensor status = made([&] { return zeros.status(values, stream); });
  const py::object rc = fn(address(indices), indices.scalar_type() == at::kLong ? 1 : 0, address(values), code,
                           indices.numel(), address(dense), dense.numel(), mode, address(ws), ws.numel(), address(status),
                           host, words, stream);
  return py::make_tuple(rc, status);
}

// Whether the lists are plain runs of one type on one device, with a value list to each index list.
bool matching_runs(const std::vector<Tensor> &indices, const std::vector<Tensor> &values) {
  if (indices.size() != values.size() || !plain_runs(indices) || !plain_runs(values)) return false;
  for (size_t i = 0; i < indices.size(); ++i)
    if (indices[i].numel() != values[i].numel() || indices[i].device() != values[i].device()) return false;
  return true;
}

py::tuple decode_lists(const py::object &fn, Zeros &zeros, const std::vector<Tensor> &indices,
                       const std::vector<Tensor> &values, int code, int64_t dense_size, const Tensor &ws, int64_t stream,
                       int64_t host, int64_t words) {
  const auto [dense, status] =
      made([&] { return Two{room(values[0], dense_size, values[0].scalar_type()), zeros.status(values[0], stream)}; });
  const Lists i(indices), v(values);
  const py::object rc = fn(i.addresses(), indices[0].scalar_type() == at::kLong ? 1 : 0, v.addresses(), code, i.counts(),
                           indices.size(), address(dense), dense_size, address(ws), ws.numel(), address(status), host, words,
                           stream);
  return py::make_tuple(rc, dense);
}

// `told`: a status word that is answered for with this call's own, of work in front of it on the stream.
py::tuple bitmaps_dense(const py::object &fn, Zeros &zeros, const std::vector<Tensor> &bitmaps,
                        const std::vector<Tensor> &values, int code, const Tensor &dict, int64_t numel, const Tensor &ws,
                        int64_t stream, int64_t host, int64_t words, const std::optional<Tensor> &told) {
  const auto [dense, status] = made([&] {
    return Two{room(values[0], numel, values[0].scalar_type()), told ? *told : zeros.status(values[0], stream)};
  });
  const Lists b(bitmaps), v(values);
  const py::object rc = fn(address(dict), numel, bitmaps.size(), b.addresses(), b.counts(), v.addresses(), code, v.counts(),
                           address(dense), address(ws), ws.numel(), address(status), host, words, stream);
  return py::make_tuple(rc, dense);
}

py::tuple bitmap_encode(const py::object &fn, Zeros &zeros, const Tensor &mapping, const Tensor &indices, const Tensor &ranks,
                        int64_t numel, int64_t count, int64_t stream, int64_t host, int64_t words) {
  const auto [bitmap, status] =
      made([&] { return Two{room(indices, std::max<int64_t>(count, 1) * 4, at::kByte), zeros.status(indices, stream)}; });
  const int idx64 = indices.scalar_type() == at::kLong ? 1 : 0;
  const py::object rc =
      host ? fn(address(mapping), mapping.numel(), address(indices), idx64, indices.numel(), py::none(), address(ranks), numel,
                address(bitmap), address(status), host, words, stream)
           : fn(address(mapping), mapping.numel(), address(indices), idx64, indices.numel(), py::none(), address(ranks), numel,
                address(bitmap), address(status), stream);
  return py::make_tuple(rc, bitmap.narrow(0, 0, (mapping.numel() + 7) / 8), status);
}

py::tuple tables(const py::object &fn, Zeros &zeros, const Tensor &input, int code, int64_t m, int64_t serial_n,
                 int64_t partitions, int rehash, int64_t stream, int64_t host, int64_t words) {
  const auto [memory, serial, offsets, status] = made([&] {
    return Four{room(input, m, at::kInt), room(input, serial_n, at::kInt), room(input, partitions, at::kInt), zeros.status(input, stream)};
  });
  const py::object rc = fn(address(input), code, input.numel(), address(memory), m, address(serial), serial_n,
                           address(offsets), partitions, rehash, address(status), host, words, stream);
  return py::make_tuple(rc, memory, serial, offsets, status);
}

py::tuple table_find(const py::object &fn, Zeros &zeros, const Tensor &memory, int64_t partitions, int64_t n, int64_t ws_bytes,
                     int64_t stream, int64_t host, int64_t words) {
  // beside the split sizes, the words in which the walk adds them up; no workspace that is kept from call to call: the
  // thread may walk another table before these lists are used up
  const auto [all, status, ws] = made([&] {
    return Three{zeros.words(memory, stream, 3 * partitions + 66), zeros.status(memory, stream), room(memory, ws_bytes, at::kByte)};
  });
  const Tensor splits = all.narrow(0, 0, partitions);
  const py::object rc =
      host ? fn(address(memory), memory.numel(), partitions, n, address(splits), address(all) + 8 * partitions, address(ws),
                ws_bytes, address(status), host, words, stream)
           : fn(address(memory), memory.numel(), partitions, n, address(splits), address(ws), ws_bytes, address(status), stream);
  return py::make_tuple(rc, splits, status, ws);
}

py::tuple table_gather(const py::object &fn, const Tensor &memory, const Tensor &flat, int code,
                       const std::vector<int64_t> &sizes, const Tensor &ws, int64_t stream) {
  int64_t total = 0;
  for (int64_t s : sizes) total += s;
  const auto [idx, val] = made([&] { return Two{room(flat, total, at::kInt), room(flat, total, flat.scalar_type())}; });
  const py::object rc = fn(address(memory), memory.numel(), sizes.size(), address(flat), code, flat.numel(), address(idx),
                           address(val), total, address(ws), ws.numel(), stream);
  return py::make_tuple(rc, at::split_with_sizes(idx, sizes), at::split_with_sizes(val, sizes));
}

// The buffers of a step (zen_encode_merge) and everything in its arguments that follows from them; `wait`: the merge's
// stream has to wait for the zeroed words.
py::tuple step_buffers(int64_t args, Zeros &zeros, const Tensor &flat, const Tensor &indices, const Tensor &values,
                       int64_t capacity, int64_t partitions, int64_t stream, int64_t merge_stream, const Tensor &ws,
                       const Tensor &merge_ws) {
  zen_encode_merge_args *a = reinterpret_cast<zen_encode_merge_args *>(args);
  const int64_t r = indices.numel();
  bool wait = false;
  // small: split sizes, merged count, the two status words
  const auto [idx, val, m_idx, m_val, small] = made([&] {
    return Five{room(flat, capacity, at::kInt), room(flat, capacity, flat.scalar_type()), room(flat, r, at::kInt),
                room(flat, r, at::kFloat),
                merge_stream ? zeros.words_for(flat, stream, partitions + 2, merge_stream, &wait)
                             : zeros.words(flat, stream, partitions + 2)};
  });
  const Tensor splits = small.narrow(0, 0, partitions), count = small.narrow(0, partitions, 1);
  const Tensor both = small.narrow(0, partitions + 1, 1).view(at::kInt);
  const Tensor status = both.narrow(0, 0, 1), m_status = both.narrow(0, 1, 1);
  a->input = flat.data_ptr();
  a->out_idx = static_cast<int32_t *>(idx.data_ptr());
  a->out_val = val.data_ptr();
  a->splits = static_cast<int64_t *>(splits.data_ptr());
  a->workspace = ws.data_ptr();
  a->workspace_bytes = (size_t)ws.numel();
  a->status = static_cast<int32_t *>(status.data_ptr());
  a->recv_idx = indices.data_ptr();
  a->recv_idx64 = indices.scalar_type() == at::kLong;
  a->recv_val = values.data_ptr();
  a->merged_idx = m_idx.data_ptr();
  a->merged_val = static_cast<float *>(m_val.data_ptr());
  a->merged_count = static_cast<int64_t *>(count.data_ptr());
  a->merge_workspace = merge_ws.data_ptr();
  a->merge_workspace_bytes = (size_t)merge_ws.numel();
  a->merge_status = static_cast<int32_t *>(m_status.data_ptr());
  a->stream = reinterpret_cast<void *>(stream);
  a->merge_stream = reinterpret_cast<void *>(merge_stream);
  return py::make_tuple(py::make_tuple(idx, val, splits, status), py::make_tuple(m_idx, m_val, count, m_status), wait);
}

// ------------------------------------------------- update.py: arguments are checked here too, in a microsecond or two

int type_of(const Tensor &t, const char *name, bool half = true, bool single = true) {
  switch (t.scalar_type()) {
    case at::kFloat:
      if (single) return ZEN_F32;
      break;
    case at::kBFloat16:
      return ZEN_BF16;
    case at::kHalf:
      if (half) return ZEN_F16;
      break;
    default:
      break;
  }
  throw py::type_error(std::string(name) + " must be " + (single ? "float32, " : "") + "bfloat16" + (half ? " or float16" : "") +
                       ", got " + c10::toString(t.scalar_type()));
}

void on_one_device(const Tensor &first, const Tensor &t) {
  if (t.device() != first.device())
    throw py::value_error("tensors on different devices: " + first.device().str() + " and " + t.device().str());
}

void on_gpu(const Tensor &t) {
  if (!t.is_cuda()) throw py::type_error("expected GPU tensors");
}

void plain(const Tensor &t, const char *name) {
  if (!t.is_contiguous()) throw std::runtime_error(std::string(name) + " must be contiguous");
}

void not_differentiated(const Tensor &t) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    throw std::runtime_error("an optimiser's step is not differentiated: call this under torch.no_grad()");
}

void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// First byte, and the byte behind the last one, of what a tensor's elements cover.
std::pair<const char *, const char *> extent(const Tensor &t) {
  if (t.numel() == 0) return {nullptr, nullptr};
  const char *first = static_cast<const char *>(t.data_ptr());
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {first, first + (last + 1) * t.element_size()};
}

// Whether two tensors may share memory.  Told apart beside plain stretches: two equally strided matrices whose rows lie between
// each other's (column ranges of one larger matrix).
bool overlap(const Tensor &a, const Tensor &b) {
  const auto [a0, a1] = extent(a);
  const auto [b0, b1] = extent(b);
  if (!(a0 < b1 && b0 < a1)) return false;
  if (a.dim() == 2 && b.dim() == 2 && a.strides() == b.strides() && a.scalar_type() == b.scalar_type()) {
    const int line = a.stride(1) == 1 ? 1 : 0;  // the dimension whose neighbours are neighbours in memory
    const int64_t step = a.stride(1 - line), size = a.element_size(), away = b0 - a0;
    if (a.stride(line) == 1 && step > 0 && away % size == 0) {
      const int64_t apart = (away / size % step + step) % step;
      if (a.size(line) <= apart && apart <= step - b.size(line)) return false;
    }
  }
  return true;
}

bool same(const Tensor &a, const Tensor &b) {
  return a.data_ptr() == b.data_ptr() && a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// Refuses a tensor to be written some of whose elements are one place in memory.
void one_place(const Tensor &t, const char *name) {
  std::vector<std::pair<int64_t, int64_t>> at;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) at.emplace_back(t.stride(d), t.size(d));
  std::sort(at.begin(), at.end());
  int64_t reach = 0;
  for (const auto &[stride, size] : at) {
    if (stride <= reach) throw py::value_error(std::string(name) + ": several elements are one place in memory");
    reach += (size - 1) * stride;
  }
}

using Dtype = std::optional<at::ScalarType>;

Tensor momentum_out(const Tensor &momentum, double mu, const Dtype &dtype, const std::optional<Tensor> &out, at::ScalarType like) {
  on_gpu(momentum);
  type_of(momentum, "momentum", false);
  plain(momentum, "momentum");
  not_differentiated(momentum);
  if (!(mu >= 0.0 && mu < std::numeric_limits<double>::infinity())) throw py::value_error("mu must be finite and not negative");
  if (!out) return made([&] { return at::empty(momentum.sizes(), momentum.options().dtype(dtype ? *dtype : like).requires_grad(false)); });
  if (dtype && out->scalar_type() != *dtype) throw py::type_error("out is not of that dtype");
  on_one_device(momentum, *out);
  not_differentiated(*out);
  plain(*out, "out");
  if (out->sizes() != momentum.sizes()) throw py::value_error("out is not of the momentum's shape");
  if (overlap(*out, momentum)) throw py::value_error("out overlaps the momentum");
  return *out;
}

py::tuple momentum(const py::object &fn, const Tensor &momentum, const Tensor &grad, double mu, bool nesterov, const Dtype &dtype,
                   const std::optional<Tensor> &given, int64_t stream) {
  on_gpu(grad);
  const int code = type_of(grad, "grad");
  const Tensor out = momentum_out(momentum, mu, dtype, given, grad.scalar_type());
  const int out_code = type_of(out, "update");
  on_one_device(momentum, grad);
  plain(grad, "grad");
  not_differentiated(grad);
  if (grad.sizes() != momentum.sizes()) throw py::value_error("grad is not of the momentum's shape");
  if (overlap(grad, momentum) || (overlap(out, grad) && !same(out, grad)))
    throw py::value_error("grad overlaps the momentum or a part of out");
  const py::object rc = fn(address(momentum), type_of(momentum, "momentum"), address(grad), code, grad.numel(), mu, nesterov ? 1 : 0,
                           address(out), out_code, stream);
  written(momentum);
  written(out);
  return py::make_tuple(rc, out);
}

// counts: none, one tensor (an element to a list), or one tensor or none to a list
// before: the status word of the call that made the lists
py::tuple momentum_lists(const py::object &fn, Zeros &zeros, const Tensor &momentum, const std::vector<Tensor> &indices,
                         const std::vector<Tensor> &values, double mu, bool nesterov, const std::optional<Tensor> &counted,
                         const std::optional<std::vector<std::optional<Tensor>>> &counts, const Dtype &dtype,
                         const std::optional<Tensor> &given, const std::optional<Tensor> &before, const py::object &workspace,
                         int64_t stream) {
  const size_t lists = indices.size();
  if (lists < 1 || lists > ZEN_MOMENTUM_LISTS_MOST || values.size() != lists)
    throw py::value_error("1 to " + std::to_string(ZEN_MOMENTUM_LISTS_MOST) + " lists, as many of indices as of values: got " +
                          std::to_string(lists) + " and " + std::to_string(values.size()));
  on_gpu(values[0]);
  const int code = type_of(values[0], "values");
  const at::ScalarType index = indices[0].scalar_type();
  if (index != at::kInt && index != at::kLong) throw py::type_error("indices must be int32 or int64");
  const Tensor out = momentum_out(momentum, mu, dtype, given, values[0].scalar_type());
  const int out_code = type_of(out, "update");
  const int64_t n = momentum.numel();
  if (n > 0x7fffffffll) throw py::value_error("momentum_update_sparse: at most 2^31 - 1 elements");
  const auto apart = [&](const Tensor &t) {
    if (overlap(t, momentum) || overlap(t, out)) throw py::value_error("momentum_update_sparse: a list overlaps the momentum or out");
  };
  for (size_t l = 0; l < lists; ++l) {
    const Tensor &i = indices[l], &v = values[l];
    on_one_device(momentum, i);
    on_one_device(momentum, v);
    plain(i, "indices");
    plain(v, "values");
    not_differentiated(v);
    if (i.scalar_type() != index || v.scalar_type() != values[0].scalar_type())
      throw py::type_error("the lists' indices, and their values, have one type");
    if (i.numel() != v.numel()) throw py::value_error("a list has as many indices as values");
    if (n == 0 && i.numel()) throw py::value_error("momentum_update_sparse: entries for an empty momentum");
    apart(i);
    apart(v);
  }
  std::vector<int64_t> count(lists, 0);
  const auto check = [&](const Tensor &c, int64_t elements) {
    on_one_device(momentum, c);
    if (c.scalar_type() != at::kLong) throw py::type_error("counts are int64");
    if (c.numel() != elements || c.dim() > 1) throw py::value_error("counts: one element to a list");
    apart(c);
  };
  if (counted) {
    check(*counted, (int64_t)lists);
    for (size_t l = 0; l < lists; ++l) count[l] = address(*counted) + 8 * (int64_t)l * (counted->dim() ? counted->stride(0) : 0);
  } else if (counts) {
    if (counts->size() != lists) throw py::value_error("counts: one to a list");
    for (size_t l = 0; l < lists; ++l)
      if ((*counts)[l]) {
        check(*(*counts)[l], 1);
        count[l] = address(*(*counts)[l]);
      }
  }
  if (before) {
    on_one_device(momentum, *before);
    if (before->scalar_type() != at::kInt) throw py::type_error("a status is int32");
    if (before->numel() != 1) throw py::value_error("a status is one element");
    apart(*before);
    const auto from = [&](const Tensor &t) { return overlap(*before, t); };
    if (std::any_of(indices.begin(), indices.end(), from) || std::any_of(values.begin(), values.end(), from))
      throw py::value_error("momentum_update_sparse: the status overlaps a list");
  }
  const Tensor status = before ? *before : made([&] { return zeros.status(momentum, stream); });
  const Lists i(indices), v(values);
  const py::object rc = fn(address(momentum), type_of(momentum, "momentum"), i.addresses(), index == at::kLong ? 1 : 0, v.addresses(),
                           code, i.counts(), reinterpret_cast<int64_t>(count.data()), lists, n, mu, nesterov ? 1 : 0, address(out),
                           out_code, workspace.is_none() ? 0 : address(workspace.cast<Tensor>()),
                           workspace.is_none() ? 0 : workspace.cast<Tensor>().numel(), address(status), stream);
  written(momentum);
  written(out);
  if (before) written(status);
  return py::make_tuple(rc, out, status);
}

// `room(bytes)` gives a workspace.
py::tuple product(const py::object &fn, const py::object &bytes_of, const py::object &room, const Tensor &a, const Tensor &b,
                  const std::optional<Tensor> &residual, double alpha, double beta, bool symmetric, const Dtype &dtype,
                  const std::optional<Tensor> &given, int64_t stream) {
  on_gpu(a);
  zen_product_args p = {};
  p.dtype = type_of(a, "a", true, false);
  on_one_device(a, b);
  not_differentiated(a);
  not_differentiated(b);
  if (b.scalar_type() != a.scalar_type()) throw py::type_error("a and b are not of one type");
  const int64_t d = a.dim();
  if ((d != 2 && d != 3) || b.dim() != d) throw py::value_error("a and b are two matrices, or two stacks of matrices");
  p.batch = d == 3 ? a.size(0) : 1;
  p.m = a.size(-2);
  p.k = a.size(-1);
  p.n = b.size(-1);
  if (b.size(-2) != p.k || (d == 3 && b.size(0) != p.batch)) throw py::value_error("these shapes have no product");
  if (symmetric && p.m != p.n) throw py::value_error("a symmetric result is square");
  std::vector<int64_t> shape = {p.m, p.n};
  if (d == 3) shape.insert(shape.begin(), p.batch);
  if (residual) {
    on_one_device(a, *residual);
    not_differentiated(*residual);
    if (residual->sizes() != at::IntArrayRef(shape)) throw py::value_error("residual is not of the product's shape");
    p.c = residual->data_ptr();
    p.c_dtype = type_of(*residual, "residual");
    p.c_rs = residual->stride(-2);
    p.c_cs = residual->stride(-1);
    p.c_batch = d == 3 ? residual->stride(0) : 0;
  }
  const Tensor out = given ? *given : made([&] {
    return at::empty(shape, a.options().dtype(dtype ? *dtype : residual ? residual->scalar_type() : a.scalar_type()).requires_grad(false));
  });
  if (given) {
    on_one_device(a, out);
    not_differentiated(out);
    if (out.sizes() != at::IntArrayRef(shape)) throw py::value_error("out is not of the product's shape");
    if (dtype && out.scalar_type() != *dtype) throw py::type_error("out is not of that dtype");
    one_place(out, "out");
    if (overlap(out, a) || overlap(out, b) || (residual && overlap(out, *residual) && !same(out, *residual)))
      throw py::value_error("out overlaps an input");
  }
  p.out_dtype = type_of(out, "the result");
  p.a = a.data_ptr();
  p.a_rs = a.stride(-2);
  p.a_cs = a.stride(-1);
  p.b = b.data_ptr();
  p.b_rs = b.stride(-2);
  p.b_cs = b.stride(-1);
  p.out = out.data_ptr();
  p.out_rs = out.stride(-2);
  p.out_cs = out.stride(-1);
  if (d == 3) {
    p.a_batch = a.stride(0);
    p.b_batch = b.stride(0);
    p.out_batch = out.stride(0);
  }
  p.alpha = (float)alpha;
  p.beta = (float)beta;
  p.symmetric = symmetric;
  p.stream = reinterpret_cast<void *>(stream);
  const int64_t args = reinterpret_cast<int64_t>(&p);
  p.workspace_bytes = bytes_of(args).cast<size_t>();
  Tensor ws;
  if (p.workspace_bytes) {
    ws = room(p.workspace_bytes).cast<Tensor>();
    p.workspace = ws.data_ptr();
  }
  const py::object rc = fn(args);
  written(out);
  return py::make_tuple(rc, out);
}

// Smaller side from which on the products' operands have 11 bits where the result is bf16.  The fewer rows there are, the less do
// their roundings average out: off by (2-norm, before the result's own rounding, which is 1.66e-3) at most 1.24e-3 from 64
// rows on, 1.6e-3 with 24, up to 5e-3 with two.  With 22 bits a call below takes a sixth longer (48 x 3000: 114 us, not 99).
constexpr int64_t kElevenBitsFrom = 64;

// Updates to outs (or weights), one zen_orthogonal call for each pair of strides among them; its first failure, or 0.
py::object orthogonal(const py::object &fn, const py::object &bytes_of, const py::object &room, const std::string &what,
                      const std::vector<Tensor> &updates, const std::vector<Tensor> &outs, int steps, double a, double b, double c,
                      double eps, bool precise, bool weights, double keep, double gain, int64_t stream) {
  const Tensor &first = updates[0];
  on_gpu(first);
  if (steps < 1) throw py::value_error(what + ": at least one step");
  if (!(eps >= 0)) throw py::value_error(what + ": eps must not be negative");
  zen_orthogonal_args p = {};
  p.update_dtype = type_of(first, "update");
  p.out_dtype = type_of(outs[0], weights ? "weight" : "out");
  std::map<std::array<int64_t, 4>, std::pair<std::vector<int64_t>, std::vector<int64_t>>> groups;
  struct Span {
    const char *from, *to;
    bool writes;
    const Tensor *t;
  };
  std::vector<Span> spans;
  for (size_t i = 0; i < updates.size(); ++i) {
    const Tensor &u = updates[i], &o = outs[i];
    on_one_device(first, u);
    on_one_device(first, o);
    not_differentiated(u);
    not_differentiated(o);
    if (u.sizes() != first.sizes() || u.scalar_type() != first.scalar_type() || o.scalar_type() != outs[0].scalar_type())
      throw py::value_error(what + ": the matrices of a call have one shape and one type");
    if (o.sizes() != u.sizes()) throw py::value_error(what + ": an update and its result are of different shapes");
    one_place(o, what.c_str());
    const auto eo = extent(o);
    spans.push_back({eo.first, eo.second, true, &o});
    if (weights || !same(u, o)) {
      const auto eu = extent(u);
      spans.push_back({eu.first, eu.second, false, &u});
    }
    auto &g = groups[{u.stride(0), u.stride(1), o.stride(0), o.stride(1)}];
    g.first.push_back(address(u));
    g.second.push_back(address(o));
  }
  if (first.numel() == 0) return py::int_(0);
  // what is written lies apart from everything else (an update may be its own result)
  std::sort(spans.begin(), spans.end(), [](const Span &x, const Span &y) { return x.from < y.from; });
  std::vector<const Span *> open;
  for (const Span &s : spans) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Span *o) { return o->to <= s.from; }), open.end());
    for (const Span *o : open)
      if ((s.writes || o->writes) && overlap(*s.t, *o->t)) throw py::value_error(what + ": a result overlaps another matrix");
    open.push_back(&s);
  }
  p.rows = first.size(0);
  p.cols = first.size(1);
  p.steps = steps;
  p.a = (float)a;
  p.b = (float)b;
  p.c = (float)c;
  p.eps = eps;
  p.precise = precise || std::min(p.rows, p.cols) < kElevenBitsFrom;
  p.weights = weights;
  p.keep = (float)keep;
  p.gain = (float)gain;
  p.stream = reinterpret_cast<void *>(stream);
  py::object rc = py::int_(0);
  for (auto &[strides, g] : groups) {
    p.count = (int64_t)g.first.size();
    p.updates = reinterpret_cast<const void *const *>(g.first.data());
    p.outs = reinterpret_cast<void *const *>(g.second.data());
    p.update_rs = strides[0];
    p.update_cs = strides[1];
    p.out_rs = strides[2];
    p.out_cs = strides[3];
    p.workspace_bytes = bytes_of(p.rows, p.cols, p.count, p.precise).cast<size_t>();
    Tensor ws;
    if (p.workspace_bytes) {  // none: the call is refused
      ws = room(p.workspace_bytes).cast<Tensor>();
      p.workspace = ws.data_ptr();
    }
    rc = fn(reinterpret_cast<int64_t>(&p));
    if (rc.cast<int>() != ZEN_OK) break;
  }
  for (const Tensor &o : outs) written(o);
  return rc;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::class_<Zeros>(m, "Zeros").def(py::init<>()).def("fresh", &Zeros::fresh);
  m.attr("ABI_VERSION") = ZEN_ABI_VERSION;
  m.def("one_buffer", &one_buffer);
  m.def("plain_runs", &plain_runs);
  m.def("cut", &cut);
  m.def("load_balance", &load_balance);
  m.def("merge", &merge);
  m.def("select_count", &select_count);
  m.def("sample_threshold", &sample_threshold);
  m.def("decode", &decode);
  m.def("matching_runs", &matching_runs);
  m.def("decode_lists", &decode_lists);
  m.def("bitmaps_dense", &bitmaps_dense);
  m.def("bitmap_encode", &bitmap_encode);
  m.def("tables", &tables);
  m.def("table_find", &table_find);
  m.def("table_gather", &table_gather);
  m.def("step_buffers", &step_buffers);
  m.def("momentum", &momentum);
  m.def("momentum_lists", &momentum_lists);
  m.def("product", &product);
  m.def("orthogonal", &orthogonal);
}
