// Python binding of the paged-cache and beam-search operators.
//
// A call of theirs on a small batch takes the GPU 2 to 10 us, less than checking
// its tensors and calling through ctypes from Python does (10 to 20 us).  So the
// checks, the outputs and the scratch are made here, and the C ABI is called
// directly.  Everything else of the package stays behind ctypes.
//
// Tensors that do not fit raise ValueError before anything is launched; a status
// of the C ABI raises NpuError with its message.  An operator runs on the device of
// its tensors, on that device's current stream; scratch comes from torch's
// allocator at each call, so calls on several streams and captured graphs share
// none.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "npu_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

// One tensor of a call on device `index` (-1: any CUDA device).
void check(const Tensor& t, const char* name, at::ScalarType type, int64_t dims, int index) {
  if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  if (t.scalar_type() != type)
    refuse(std::string(name) + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
  if (dims >= 0 && t.dim() != dims)
    refuse(std::string(name) + " must have " + std::to_string(dims) + " dims, got " + shape_of(t));
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
  if (index >= 0 && t.get_device() != index)
    refuse(std::string(name) + " is on cuda:" + std::to_string(t.get_device()) + ", not on cuda:" +
           std::to_string(index));
}

int device_of(const Tensor& t, const char* name) {
  if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  return t.get_device();
}

int whole(int64_t x, const char* name) {
  if (x < INT32_MIN || x > INT32_MAX) refuse(std::string(name) + " " + std::to_string(x) + " is out of range");
  return static_cast<int>(x);
}

void* stream_of(int index) { return at::cuda::getCurrentCUDAStream(index).stream(); }

void status(int rc) {
  if (rc == NPU_B200_OK) return;
  const std::string message = npu_b200_last_error();
  const py::object error = py::module_::import("llm_compiler_3_b200._native").attr("NpuError");
  PyErr_SetObject(error.ptr(), error(rc, message).ptr());
  throw py::error_already_set();
}

// A new tensor on t's device, past torch's dispatcher (a call with five of them 9.1 ->
// 7.8 us).
Tensor like(const Tensor& t, at::IntArrayRef size, at::ScalarType type) {
  return at::detail::empty_cuda(size, type, t.device(), std::nullopt);
}

Tensor output(const Tensor& t, const Maybe& out, int index) {
  if (!out) return like(t, t.sizes(), t.scalar_type());
  check(*out, "out", t.scalar_type(), -1, index);
  if (out->sizes() != t.sizes()) refuse("out must be " + shape_of(t) + ", got " + shape_of(*out));
  return *out;
}

void check_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, int64_t batch,
                 int64_t head_dim, int index) {
  check(k_pages, "k_pages", at::kHalf, 4, index);
  check(v_pages, "v_pages", at::kHalf, 4, index);
  check(table, "page_table", at::kInt, 2, index);
  if (v_pages.sizes() != k_pages.sizes() || k_pages.size(3) != head_dim)
    refuse("k_pages " + shape_of(k_pages) + ", v_pages " + shape_of(v_pages) + " and head_dim " +
           std::to_string(head_dim) + " disagree");
  if (table.size(0) != batch) refuse("page_table must have one row per sequence");
}

void check_counts(const Tensor& t, const char* name, int64_t n, int index) {
  check(t, name, at::kInt, 1, index);
  if (t.size(0) != n) refuse(std::string(name) + " must have one entry per sequence");
}

const int32_t* ints(const Tensor& t) { return t.const_data_ptr<int32_t>(); }
const int32_t* ints(const Maybe& t) { return t ? ints(*t) : nullptr; }

float scale_of(const std::optional<double>& scale, int64_t head_dim) {
  return static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(head_dim)));
}

Tensor paged_decode(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                    const Tensor& seq_lens, int64_t window, int64_t sinks, std::optional<double> scale,
                    const Maybe& out) {
  const int index = device_of(q, "q");
  check(q, "q", at::kHalf, 3, index);
  check_pages(k_pages, v_pages, table, q.size(0), q.size(2), index);
  check_counts(seq_lens, "seq_lens", q.size(0), index);
  const c10::cuda::CUDAGuard guard(index);
  Tensor o = output(q, out, index);
  const int heads = whole(q.size(1), "heads"), kv_heads = whole(k_pages.size(1), "kv_heads"),
            dim = whole(q.size(2), "head_dim");
  const size_t bytes = npu_b200_paged_decode_workspace_size(heads, kv_heads, dim);
  const Tensor scratch = like(q, {static_cast<int64_t>(bytes)}, at::kByte);
  status(npu_b200_paged_decode(
      q.const_data_ptr(), k_pages.const_data_ptr(), v_pages.const_data_ptr(), ints(table), ints(seq_lens),
      o.mutable_data_ptr(), whole(q.size(0), "batch"), heads, kv_heads, dim,
      whole(k_pages.size(0), "num_pages"), whole(k_pages.size(2), "page_size"),
      whole(table.size(1), "table entries"), whole(window, "window"), whole(sinks, "sinks"),
      scale_of(scale, dim), scratch.mutable_data_ptr(), bytes, stream_of(index)));
  return o;
}

Tensor paged_prefill(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                     const Tensor& seq_lens, const Maybe& q_lens, int64_t window, int64_t sinks,
                     std::optional<double> scale, const Maybe& out) {
  const int index = device_of(q, "q");
  check(q, "q", at::kHalf, 4, index);
  check_pages(k_pages, v_pages, table, q.size(0), q.size(3), index);
  check_counts(seq_lens, "seq_lens", q.size(0), index);
  if (q_lens) check_counts(*q_lens, "q_lens", q.size(0), index);
  const c10::cuda::CUDAGuard guard(index);
  Tensor o = output(q, out, index);
  status(npu_b200_paged_prefill(
      q.const_data_ptr(), k_pages.const_data_ptr(), v_pages.const_data_ptr(), ints(table), ints(seq_lens),
      ints(q_lens), o.mutable_data_ptr(), whole(q.size(0), "batch"), whole(q.size(1), "heads"),
      whole(k_pages.size(1), "kv_heads"), whole(q.size(3), "head_dim"), whole(q.size(2), "queries"),
      whole(k_pages.size(0), "num_pages"), whole(k_pages.size(2), "page_size"),
      whole(table.size(1), "table entries"), whole(window, "window"), whole(sinks, "sinks"),
      scale_of(scale, q.size(3)), stream_of(index)));
  return o;
}

void paged_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                  const Tensor& table, const Tensor& starts, const Maybe& lens) {
  const int index = device_of(k, "k");
  check(k, "k", at::kHalf, 4, index);
  check(v, "v", at::kHalf, 4, index);
  if (v.sizes() != k.sizes()) refuse("k and v must have one shape");
  check_pages(k_pages, v_pages, table, k.size(0), k.size(3), index);
  if (k_pages.size(1) != k.size(1))
    refuse("k has " + std::to_string(k.size(1)) + " heads but the pages " + std::to_string(k_pages.size(1)));
  check_counts(starts, "starts", k.size(0), index);
  if (lens) check_counts(*lens, "lens", k.size(0), index);
  const c10::cuda::CUDAGuard guard(index);
  status(npu_b200_paged_append(
      k.const_data_ptr(), v.const_data_ptr(), k_pages.mutable_data_ptr(), v_pages.mutable_data_ptr(),
      ints(table), ints(starts), ints(lens), whole(k.size(0), "batch"), whole(k.size(1), "heads"),
      whole(k.size(2), "rows"), whole(k.size(3), "head_dim"), whole(k_pages.size(0), "num_pages"),
      whole(k_pages.size(2), "page_size"), whole(table.size(1), "table entries"), stream_of(index)));
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> page_update(const Tensor& table, const Tensor& seq_lens,
                                                              const Tensor& parents, const Tensor& capacity,
                                                              const Tensor& refs, int64_t page_size) {
  const int index = device_of(table, "page_table");
  check(table, "page_table", at::kInt, 2, index);
  check(refs, "page_refs", at::kInt, 1, index);
  check(parents, "parents", at::kInt, 1, index);
  check_counts(seq_lens, "seq_lens", table.size(0), index);
  check_counts(capacity, "capacity", parents.size(0), index);
  const c10::cuda::CUDAGuard guard(index);
  const int64_t rows = parents.size(0), entries = table.size(1), pages = refs.size(0);
  Tensor new_table = like(table, {rows, entries}, at::kInt), lens = like(table, {rows}, at::kInt);
  Tensor new_refs = like(table, {pages}, at::kInt), copies = like(table, {2, rows}, at::kInt);
  Tensor info = like(table, {3}, at::kInt);
  status(npu_b200_page_update(
      ints(table), ints(seq_lens), ints(parents), ints(capacity), ints(refs),
      new_table.mutable_data_ptr<int32_t>(), lens.mutable_data_ptr<int32_t>(),
      new_refs.mutable_data_ptr<int32_t>(), copies.mutable_data_ptr<int32_t>(),
      info.mutable_data_ptr<int32_t>(), whole(table.size(0), "rows"), whole(rows, "rows"),
      whole(entries, "table entries"), whole(page_size, "page_size"), whole(pages, "pages"),
      stream_of(index)));
  return {new_table, lens, new_refs, copies, info};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> page_compact(const Tensor& table, const Tensor& refs) {
  const int index = device_of(table, "page_table");
  check(table, "page_table", at::kInt, 2, index);
  check(refs, "page_refs", at::kInt, 1, index);
  const c10::cuda::CUDAGuard guard(index);
  const int64_t pages = refs.size(0);
  Tensor new_table = like(table, table.sizes(), at::kInt), new_refs = like(table, {pages}, at::kInt);
  Tensor moves = like(table, {2, pages / 2 > 0 ? pages / 2 : 1}, at::kInt);
  Tensor where = like(table, {pages}, at::kInt), info = like(table, {2}, at::kInt);
  status(npu_b200_page_compact(
      ints(table), ints(refs), new_table.mutable_data_ptr<int32_t>(), new_refs.mutable_data_ptr<int32_t>(),
      moves.mutable_data_ptr<int32_t>(), where.mutable_data_ptr<int32_t>(), info.mutable_data_ptr<int32_t>(),
      whole(table.size(0), "rows"), whole(table.size(1), "table entries"), whole(pages, "pages"),
      stream_of(index)));
  return {new_table, new_refs, moves, where, info};
}

void page_copy(const Tensor& pool, const Tensor& pages, const Maybe& count) {
  const int index = device_of(pool, "pool");
  if (!pool.is_contiguous() || pool.dim() < 3 || pool.numel() == 0)
    refuse("pool must be a contiguous [slabs, pages, ...], got " + shape_of(pool));
  check(pages, "pages", at::kInt, 2, index);
  if (pages.size(0) != 2) refuse("pages must be [2, n]: from and to");
  if (count) {
    check(*count, "count", at::kInt, 1, index);
    if (count->size(0) < 1) refuse("count must hold a number");
  }
  const c10::cuda::CUDAGuard guard(index);
  const int64_t slabs = pool.size(0), n = pool.size(1);
  status(npu_b200_page_copy(pool.mutable_data_ptr(), ints(pages), ints(count), whole(pages.size(1), "copies"),
                            whole(slabs, "slabs"), whole(n, "pages"),
                            static_cast<size_t>(pool.numel() / (slabs * n) * pool.element_size()),
                            stream_of(index)));
}

std::tuple<Tensor, Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores,
                                                      int64_t width, const Maybe& done, int64_t eos) {
  const int index = device_of(logits, "logits");
  const bool f32 = logits.scalar_type() == at::kFloat;
  if (!f32 && logits.scalar_type() != at::kHalf)
    refuse(std::string("logits must be float16 or float32, got ") + c10::toString(logits.scalar_type()));
  check(logits, "logits", logits.scalar_type(), 3, index);
  check(scores, "scores", at::kFloat, 2, index);
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  if (scores.size(0) != batch || scores.size(1) != beams)
    refuse("scores must be [batch, beams] of the logits, got " + shape_of(scores));
  if (done) {
    check(*done, "done", at::kBool, 2, index);
    if (done->sizes() != scores.sizes()) refuse("done must have the shape of scores");
  }
  if (width < 1) refuse("width must be positive, got " + std::to_string(width));
  const int b = whole(batch, "batch"), w = whole(beams, "beams"), v = whole(vocab, "vocab"),
            n = whole(width, "width");
  const c10::cuda::CUDAGuard guard(index);
  Tensor best = like(logits, {batch, width}, at::kFloat), tokens = like(logits, {batch, width}, at::kInt);
  Tensor parents = like(logits, {batch, width}, at::kInt), ended = like(logits, {batch, width}, at::kBool);
  const size_t bytes = npu_b200_beam_select_workspace_size(b, w, v, n);
  const Tensor scratch = like(logits, {static_cast<int64_t>(bytes)}, at::kByte);
  status(npu_b200_beam_select(
      logits.const_data_ptr(), f32, scores.const_data_ptr<float>(),
      done ? static_cast<const uint8_t*>(done->const_data_ptr()) : nullptr, best.mutable_data_ptr<float>(),
      tokens.mutable_data_ptr<int32_t>(), parents.mutable_data_ptr<int32_t>(),
      static_cast<uint8_t*>(ended.mutable_data_ptr()), b, w, v, n, whole(eos, "eos"),
      scratch.mutable_data_ptr(), bytes, stream_of(index)));
  return {best, tokens, parents, ended};
}

Tensor beam_reorder(const Tensor& state, const Tensor& parents, const Maybe& out) {
  const int index = device_of(state, "state");
  if (!state.is_contiguous() || state.dim() < 1 || state.numel() == 0)
    refuse("state must be a contiguous [rows, ...], got " + shape_of(state));
  check(parents, "parents", at::kInt, -1, index);
  std::vector<int64_t> size = state.sizes().vec();
  const int64_t rows = size[0];
  size[0] = parents.numel();
  const c10::cuda::CUDAGuard guard(index);
  if (out) {
    check(*out, "out", state.scalar_type(), -1, index);
    if (out->sizes() != at::IntArrayRef(size)) refuse("out must have a row for each parent, got " + shape_of(*out));
  }
  Tensor o = out ? *out : like(state, size, state.scalar_type());
  status(npu_b200_beam_reorder(state.const_data_ptr(), ints(parents), o.mutable_data_ptr(), whole(rows, "rows"),
                               whole(size[0], "rows"),
                               static_cast<size_t>(state.numel() / rows * state.element_size()),
                               stream_of(index)));
  return o;
}

}  // namespace

PYBIND11_MODULE(_bindings, m) {
  py::register_exception_translator([](std::exception_ptr p) {  // torch's own types for its errors
    try {
      if (p) std::rethrow_exception(p);
    } catch (const c10::OutOfMemoryError& e) {
      PyErr_SetString(py::module_::import("torch").attr("OutOfMemoryError").ptr(), e.what_without_backtrace());
    }
  });
  m.attr("built_for") = NPU_B200_BUILT_FOR;  // the version of torch
  m.def("paged_decode", &paged_decode);
  m.def("paged_prefill", &paged_prefill);
  m.def("paged_append", &paged_append);
  m.def("page_update", &page_update);
  m.def("page_compact", &page_compact);
  m.def("page_copy", &page_copy);
  m.def("beam_select", &beam_select);
  m.def("beam_reorder", &beam_reorder);
}
