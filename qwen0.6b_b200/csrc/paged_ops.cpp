// paged_C: PyTorch extension module behind paged.py, the operators on paged KV
// pools.  The kernels and their C ABI live in libqwen_b200.so
// (include/qwen_b200_paged.h); this file checks tensors and allocates the
// outputs.  Bad arguments raise ValueError, failed launches RuntimeError.
// (Through ctypes the same checks in Python took 41 us per attention call,
// three times its time on the device.)
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>
#include <vector>

#include "qwen_b200.h"
#include "qwen_b200_paged.h"

namespace {

namespace py = pybind11;
using torch::Tensor;

void check_rc(int rc, const char *what) {
  if (rc == 0) return;
  char msg[512];
  qwen_b200_last_error(msg, sizeof(msg));
  // Codes of the C ABI that name a bad argument; the others are launch failures.
  const bool argument = rc == 10 || rc == 11 || rc == 13 || rc == 14 || rc == 15;
  TORCH_CHECK_VALUE(!argument, what, " failed (code ", rc, "): ", msg);
  TORCH_CHECK(false, what, " failed (code ", rc, "): ", msg);
}

void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

QwenPagePools pools_of(const Tensor &k, const Tensor &v) {
  for (const Tensor *t : {&k, &v})
    TORCH_CHECK_VALUE(t->is_cuda() && t->dim() >= 3 && t->is_contiguous() && t->numel() > 0,
                      t == &k ? "k_pool" : "v_pool",
                      " must be a contiguous, non-empty CUDA tensor [num_pages, ..., page_tokens, dim]");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == v.device(),
                    "k_pool and v_pool must have the same shape, type and device");
  const int64_t n = k.size(0), tokens = k.size(-2), bytes = k.size(-1) * k.element_size();
  const int64_t inner = k.numel() / (n * tokens * k.size(-1));
  TORCH_CHECK_VALUE(n < (1ll << 31) && tokens < (1ll << 31) && bytes < (1ll << 31) && inner < (1ll << 31),
                    "pool dimensions over 2^31");
  return QwenPagePools{k.data_ptr(), v.data_ptr(), static_cast<int>(n), static_cast<int>(inner),
                       static_cast<int>(tokens), static_cast<int>(bytes)};
}

QwenPageTable table_of(const Tensor &t) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.dim() == 2 && t.scalar_type() == torch::kInt && t.numel() > 0 &&
                        (t.stride(1) == 1 || t.size(1) == 1),
                    "page_table must be a CUDA int32 tensor [num_seqs, max_pages] with contiguous rows");
  TORCH_CHECK_VALUE(t.size(0) < (1ll << 31) && t.size(1) < (1ll << 31), "page_table dimensions over 2^31");
  return QwenPageTable{t.data_ptr<int>(), static_cast<int>(t.size(0)), static_cast<int>(t.size(1)),
                       t.size(0) > 1 ? t.stride(0) : t.size(1)};
}

// A list of integers on the host, as contiguous int32: any Python iterable of
// integers, or a tensor.  (Lists are read here: through torch.tensor a copy of
// one page took 7.7 us on the host, 3.1 now, of 255 pages 50 and 17.)
class HostList {
 public:
  HostList(const py::object &given, const char *name, int64_t n = -1) {
    if (THPVariable_Check(given.ptr()))
      read(THPVariable_Unpack(given.ptr()), name);
    else
      read(given, name);
    TORCH_CHECK_VALUE(n < 0 || n_ == n, name, " has ", n_, " entries, the other lists ", n);
    TORCH_CHECK_VALUE(n_ < (1ll << 31), name, " has over 2^31 entries");
  }
  const int *data() const { return data_; }
  int size() const { return static_cast<int>(n_); }

 private:
  void read(const Tensor &t, const char *name) {
    TORCH_CHECK_VALUE(t.device().is_cpu() && t.dim() == 1 && at::isIntegralType(t.scalar_type(), false), name,
                      " must be a one-dimensional list of integers on the host");
    t_ = t;
    if (t.scalar_type() != torch::kInt) {
      const Tensor wide = t.to(torch::kLong);
      TORCH_CHECK_VALUE(wide.numel() == 0 || (wide.min().item<int64_t>() >= -(1ll << 31) &&
                                              wide.max().item<int64_t>() < (1ll << 31)),
                        name, " holds a value outside 32 bits");
      t_ = wide.to(torch::kInt);
    }
    t_ = t_.contiguous();
    data_ = t_.data_ptr<int>();
    n_ = t_.numel();
  }
  void read(const py::object &given, const char *name) {
    const auto seq = py::reinterpret_steal<py::object>(PySequence_Fast(given.ptr(), ""));
    if (!seq) PyErr_Clear();
    TORCH_CHECK_VALUE(seq, name, " must be a one-dimensional list of integers on the host");
    n_ = PySequence_Fast_GET_SIZE(seq.ptr());
    v_.resize(n_);
    for (int64_t i = 0; i < n_; ++i) {
      // (A new reference: an item's __index__ may change the list.)
      const auto item = py::reinterpret_borrow<py::object>(i < PySequence_Fast_GET_SIZE(seq.ptr())
                                                               ? PySequence_Fast_GET_ITEM(seq.ptr(), i)
                                                               : Py_None);
      const auto x = py::reinterpret_steal<py::object>(PyNumber_Index(item.ptr()));
      if (!x) PyErr_Clear();
      TORCH_CHECK_VALUE(x, name, " must be a one-dimensional list of integers on the host");
      int over = 0;
      const long long value = PyLong_AsLongLongAndOverflow(x.ptr(), &over);
      TORCH_CHECK_VALUE(over == 0 && value >= -(1ll << 31) && value < (1ll << 31), name,
                        " holds a value outside 32 bits");
      v_[i] = static_cast<int>(value);
    }
    data_ = v_.data();
  }
  Tensor t_;
  std::vector<int> v_;
  const int *data_ = nullptr;
  int64_t n_ = 0;
};

void same_device(const Tensor &t, const Tensor &k) {
  TORCH_CHECK_VALUE(t.device() == k.device(), "page_table is on ", t.device(), ", the pools on ", k.device());
}

void copy_pages(const Tensor &k, const Tensor &v, const py::object &src, const py::object &dst,
                const py::object &tokens) {
  const QwenPagePools p = pools_of(k, v);
  const HostList s(src, "src"), d(dst, "dst", s.size());
  std::optional<HostList> t;
  if (!tokens.is_none()) t.emplace(tokens, "tokens", s.size());
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(qwen_b200_pages_copy(&p, s.data(), d.data(), t ? t->data() : nullptr, s.size(), stream_of(k)), "copy_pages");
}

void fork_pages(const Tensor &table, const Tensor &k, const Tensor &v, const py::object &parents,
                const py::object &children, const py::object &lengths, const py::object &new_pages) {
  const QwenPagePools p = pools_of(k, v);
  const QwenPageTable t = table_of(table);
  same_device(table, k);
  const HostList from(parents, "parents"), to(children, "children", from.size()), n(lengths, "lengths", from.size()),
      pages(new_pages, "new_pages", from.size());
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(qwen_b200_pages_fork(&p, &t, from.data(), to.data(), n.data(), pages.data(), from.size(), stream_of(k)),
           "fork_pages");
}

void compact_pages(const Tensor &table, const Tensor &k, const Tensor &v, const py::object &src,
                   const py::object &dst) {
  const QwenPagePools p = pools_of(k, v);
  const QwenPageTable t = table_of(table);
  same_device(table, k);
  const HostList s(src, "src"), d(dst, "dst", s.size());
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(qwen_b200_pages_compact(&p, &t, s.data(), d.data(), s.size(), stream_of(k)), "compact_pages");
}

void free_pages(const Tensor &table, const py::object &seqs) {
  const QwenPageTable t = table_of(table);
  const HostList s(seqs, "seqs");
  const c10::cuda::CUDAGuard guard(table.device());
  check_rc(qwen_b200_pages_free(&t, s.data(), s.size(), stream_of(table)), "free_pages");
}

// Stride of a dimension; that of a one-element dimension, which torch leaves
// arbitrary, as in a contiguous tensor.
int64_t stride_of(const Tensor &t, int64_t d) {
  if (t.size(d) > 1) return t.stride(d);
  int64_t s = 1;
  for (int64_t i = d + 1; i < t.dim(); ++i) s *= t.size(i);
  return s;
}

std::tuple<Tensor, std::optional<Tensor>> prefix_attention(
    const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &seq_ids,
    const Tensor &lengths, const Tensor &header, const Tensor &words, int64_t max_length, int64_t workspace_bytes,
    std::optional<double> scale, const std::optional<Tensor> &out_, bool return_lse) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 4 && v.dim() == 4, "q must have 3 dimensions, the pools 4");
  const auto type = q.scalar_type();
  TORCH_CHECK_VALUE(type == torch::kHalf || type == torch::kBFloat16, "q must be an fp16 or bf16 tensor, got ", type);
  TORCH_CHECK_VALUE(q.is_cuda() && q.device() == words.device(), "q is on ", q.device(), ", the plan on ",
                    words.device());
  for (const Tensor *t : {&k, &v})
    TORCH_CHECK_VALUE(t->scalar_type() == type && t->device() == q.device(), "pools of ", t->scalar_type(), " on ",
                      t->device(), ", q is ", type, " on ", q.device());
  const int *h = header.data_ptr<int>();
  const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k_pool and v_pool must have the same shape");
  for (int d = 0; d < 3; ++d)
    TORCH_CHECK_VALUE(stride_of(k, d) == stride_of(v, d), "k_pool and v_pool must have the same strides");
  TORCH_CHECK_VALUE(k.size(3) == dim, "pools of dim ", k.size(3), ", q of dim ", dim);
  TORCH_CHECK_VALUE(k.size(0) < (1ll << 31) && k.size(2) < (1ll << 31) && k.numel() > 0, "pool dimensions");
  const QwenPageTable t = table_of(table);
  TORCH_CHECK_VALUE(table.device() == q.device(), "page_table is on ", table.device(), ", q on ", q.device());
  for (const Tensor *x : {&seq_ids, &lengths})
    TORCH_CHECK_VALUE(x->scalar_type() == torch::kInt && x->dim() == 1 && x->size(0) == rows && x->is_contiguous() &&
                          x->device() == q.device(),
                      x == &lengths ? "lengths" : "seq_ids", " must be a contiguous int32 tensor [", rows, "] on ",
                      q.device());
  const c10::cuda::CUDAGuard guard(q.device());
  // A plan may be dropped while calls on other streams than its own still read it.
  c10::cuda::CUDACachingAllocator::recordStream(words.storage().data_ptr(),
                                                c10::cuda::getCurrentCUDAStream(q.device().index()));
  Tensor out;
  if (out_) {
    out = *out_;
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == type && out.device() == q.device(),
                      "out must have q's shape, type and device");
    for (const Tensor *t : {&q, &k, &v})
      TORCH_CHECK_VALUE(at::get_overlap_status(out, *t) != at::MemOverlapStatus::Partial &&
                            (t == &q || at::get_overlap_status(out, *t) != at::MemOverlapStatus::Full),
                        "out overlaps ", t == &q ? "q (it may be q itself)" : "the pools");
    // One of rows and heads lies within a step of the other.
    const int64_t sr = out.size(0) > 1 ? out.stride(0) : 1ll << 60, sh = out.size(1) > 1 ? out.stride(1) : 1ll << 60;
    const int64_t inner = sr < sh ? sr : sh, n = sr < sh ? out.size(0) : out.size(1);
    TORCH_CHECK_VALUE(inner >= dim && (sr < sh ? sh : sr) >= inner * (n - 1) + dim, "out's rows or heads overlap");
  } else {
    out = torch::empty({rows, heads, dim}, q.options());
  }
  for (const Tensor *x : {&q, &k, &v, const_cast<const Tensor *>(&out)})
    TORCH_CHECK_VALUE(x->size(-1) == 1 || x->stride(-1) == 1, "the last dimension must be contiguous");
  std::optional<Tensor> lse;
  if (return_lse) lse = torch::empty({rows, heads}, q.options().dtype(torch::kFloat));
  // The workspace comes from the caching allocator with each call: calls on
  // several streams, or captured into several graphs, have one each.
  const Tensor ws = torch::empty({workspace_bytes}, q.options().dtype(torch::kByte));
  QwenPrefixAttention a{};
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.k_pool = k.data_ptr();
  a.v_pool = v.data_ptr();
  a.page_table = t.entries;
  a.seq_ids = seq_ids.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.plan_header = h;
  a.plan = words.data_ptr<int>();
  a.workspace = ws.data_ptr();
  a.workspace_bytes = workspace_bytes;
  a.q_row_stride = stride_of(q, 0);
  a.q_head_stride = stride_of(q, 1);
  a.out_row_stride = stride_of(out, 0);
  a.out_head_stride = stride_of(out, 1);
  a.page_stride = stride_of(k, 0);
  a.head_stride = stride_of(k, 1);
  a.token_stride = stride_of(k, 2);
  a.table_pitch = t.pitch;
  a.rows = static_cast<int>(rows);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(k.size(1));
  a.dim = static_cast<int>(dim);
  a.dtype = type == torch::kBFloat16;
  a.num_pages = static_cast<int>(k.size(0));
  a.page_tokens = static_cast<int>(k.size(2));
  a.num_seqs = t.num_seqs;
  a.max_pages = t.max_pages;
  a.max_length = static_cast<int>(max_length);
  a.scale = scale ? static_cast<float>(*scale) : static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
  check_rc(qwen_b200_prefix_attention(&a, stream_of(q)), "shared_prefix_attention");
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("copy_pages", &copy_pages);
  m.def("fork_pages", &fork_pages);
  m.def("compact_pages", &compact_pages);
  m.def("free_pages", &free_pages);
  m.def("prefix_attention", &prefix_attention);
}
