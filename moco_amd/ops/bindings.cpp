// Python <-> HIP bindings for moco_amd._C.
// This is the only torch-dependent TU; the kernels live in hip/*.hip behind
// the C ABI of hip/launchers.h.
#include <torch/extension.h>

#include <ATen/FuncTorchTLS.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <cmath>

#include "hip/launchers.h"

namespace {

void* cur_stream() {
  return (void*)at::cuda::getCurrentCUDAStream().stream();
}

#define CHECK_LAUNCH(expr)                                            \
  do {                                                                \
    int rc_ = (expr);                                                 \
    TORCH_CHECK(rc_ == 0, #expr " failed with hipError_t=", rc_);     \
  } while (0)

#define CHECK_CUDA_CONTIG(t)                                          \
  TORCH_CHECK((t).is_cuda() && (t).is_contiguous(), #t,               \
              " must be a contiguous GPU tensor")

bool is_bf16(const torch::Tensor& t) {
  return t.scalar_type() == torch::kBFloat16;
}

// ---------------------------------------------------------------------------
std::vector<torch::Tensor> l2norm_rows_fwd(torch::Tensor x) {
  CHECK_CUDA_CONTIG(x);
  TORCH_CHECK(x.dim() == 2, "x must be [N, C]");
  TORCH_CHECK(is_bf16(x) || x.scalar_type() == torch::kFloat32);
  at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty_like(x);
  auto inv_norm = torch::empty({x.size(0)},
                               x.options().dtype(torch::kFloat32));
  CHECK_LAUNCH(launch_l2norm_fwd(cur_stream(), x.data_ptr(), y.data_ptr(),
                                 inv_norm.data_ptr<float>(), x.size(0),
                                 x.size(1), is_bf16(x)));
  return {y, inv_norm};
}

torch::Tensor l2norm_rows_bwd(torch::Tensor g, torch::Tensor y,
                              torch::Tensor inv_norm) {
  CHECK_CUDA_CONTIG(g);
  CHECK_CUDA_CONTIG(y);
  TORCH_CHECK(g.sizes() == y.sizes() && g.scalar_type() == y.scalar_type());
  at::cuda::CUDAGuard guard(g.device());
  auto gx = torch::empty_like(g);
  CHECK_LAUNCH(launch_l2norm_bwd(cur_stream(), g.data_ptr(), y.data_ptr(),
                                 inv_norm.data_ptr<float>(), gx.data_ptr(),
                                 g.size(0), g.size(1), is_bf16(g)));
  return gx;
}

// ---------------------------------------------------------------------------
torch::Tensor contrastive_fwd(torch::Tensor q, torch::Tensor k,
                              torch::Tensor queue_kc, double invT) {
  CHECK_CUDA_CONTIG(q);
  CHECK_CUDA_CONTIG(k);
  CHECK_CUDA_CONTIG(queue_kc);
  TORCH_CHECK(is_bf16(q) && is_bf16(k) && is_bf16(queue_kc),
              "contrastive_fwd expects bf16 q/k/queue_kc");
  const int64_t N = q.size(0), C = q.size(1), K = queue_kc.size(0);
  TORCH_CHECK(k.size(0) == N && k.size(1) == C && queue_kc.size(1) == C);
  at::cuda::CUDAGuard guard(q.device());
  auto out = torch::empty({N, 1 + K}, q.options().dtype(torch::kFloat32));
  CHECK_LAUNCH(launch_contrastive_fwd(cur_stream(), q.data_ptr(),
                                      k.data_ptr(), queue_kc.data_ptr(),
                                      out.data_ptr<float>(), N, C, K,
                                      (float)invT));
  return out;
}

torch::Tensor contrastive_bwd(torch::Tensor g, torch::Tensor k,
                              torch::Tensor queue_ck, double invT) {
  CHECK_CUDA_CONTIG(g);
  CHECK_CUDA_CONTIG(k);
  CHECK_CUDA_CONTIG(queue_ck);
  TORCH_CHECK(g.scalar_type() == torch::kFloat32 &&
              queue_ck.scalar_type() == torch::kFloat32 && is_bf16(k));
  const int64_t N = g.size(0), C = queue_ck.size(0), K = queue_ck.size(1);
  TORCH_CHECK(g.size(1) == 1 + K && k.size(0) == N && k.size(1) == C);
  at::cuda::CUDAGuard guard(g.device());
  auto dq = torch::zeros({N, C}, g.options());
  CHECK_LAUNCH(launch_contrastive_bwd(cur_stream(), g.data_ptr<float>(),
                                      k.data_ptr(),
                                      queue_ck.data_ptr<float>(),
                                      dq.data_ptr<float>(), N, C, K,
                                      (float)invT));
  return dq;
}

// ---------------------------------------------------------------------------
std::vector<torch::Tensor> softmax_ce0_fwd(torch::Tensor logits) {
  CHECK_CUDA_CONTIG(logits);
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 && logits.dim() == 2);
  at::cuda::CUDAGuard guard(logits.device());
  const int64_t N = logits.size(0), M = logits.size(1);
  auto opts = logits.options();
  auto loss_rows = torch::empty({N}, opts);
  auto row_max = torch::empty({N}, opts);
  auto row_lse = torch::empty({N}, opts);
  CHECK_LAUNCH(launch_softmax_ce0_fwd(
      cur_stream(), logits.data_ptr<float>(), loss_rows.data_ptr<float>(),
      row_max.data_ptr<float>(), row_lse.data_ptr<float>(), N, M));
  return {loss_rows, row_max, row_lse};
}

// gscale (optional fp32 scalar tensor): extra scale read on device — the
// upstream grad under hipGraph capture, where a host .item() would sync
torch::Tensor softmax_ce0_bwd(torch::Tensor logits, torch::Tensor row_max,
                              torch::Tensor row_lse, double scale,
                              c10::optional<torch::Tensor> gscale) {
  CHECK_CUDA_CONTIG(logits);
  at::cuda::CUDAGuard guard(logits.device());
  auto dlogits = torch::empty_like(logits);
  const float* gs = nullptr;
  if (gscale.has_value()) {
    TORCH_CHECK(gscale->is_cuda() &&
                gscale->scalar_type() == torch::kFloat32 &&
                gscale->numel() == 1);
    gs = gscale->data_ptr<float>();
  }
  CHECK_LAUNCH(launch_softmax_ce0_bwd(
      cur_stream(), logits.data_ptr<float>(), row_max.data_ptr<float>(),
      row_lse.data_ptr<float>(), dlogits.data_ptr<float>(), (float)scale,
      gs, logits.size(0), logits.size(1)));
  return dlogits;
}

// ---------------------------------------------------------------------------
// graph-replay-safe enqueue: ring position read/advanced from the queue_ptr
// buffer on device (a host ptr would be frozen into a captured graph)
void queue_enqueue_dev(torch::Tensor queue,
                       c10::optional<torch::Tensor> queue_kc,
                       torch::Tensor keys, torch::Tensor queue_ptr) {
  CHECK_CUDA_CONTIG(queue);
  CHECK_CUDA_CONTIG(keys);
  TORCH_CHECK(queue.scalar_type() == torch::kFloat32);
  TORCH_CHECK(queue_ptr.is_cuda() &&
              queue_ptr.scalar_type() == torch::kInt64);
  const int64_t C = queue.size(0), K = queue.size(1), B = keys.size(0);
  TORCH_CHECK(keys.size(1) == C && K % B == 0);
  void* kc = nullptr;
  if (queue_kc.has_value()) {
    CHECK_CUDA_CONTIG(*queue_kc);
    TORCH_CHECK(is_bf16(*queue_kc) && queue_kc->size(0) == K &&
                queue_kc->size(1) == C);
    kc = queue_kc->data_ptr();
  }
  at::cuda::CUDAGuard guard(queue.device());
  CHECK_LAUNCH(launch_queue_enqueue_dev(
      cur_stream(), queue.data_ptr<float>(), kc, keys.data_ptr(),
      is_bf16(keys), C, K, B, queue_ptr.data_ptr<int64_t>()));
}

void queue_enqueue(torch::Tensor queue, c10::optional<torch::Tensor> queue_kc,
                   torch::Tensor keys, int64_t ptr) {
  CHECK_CUDA_CONTIG(queue);
  CHECK_CUDA_CONTIG(keys);
  TORCH_CHECK(queue.scalar_type() == torch::kFloat32);
  const int64_t C = queue.size(0), K = queue.size(1), B = keys.size(0);
  TORCH_CHECK(keys.size(1) == C && ptr + B <= K);
  void* kc = nullptr;
  if (queue_kc.has_value()) {
    CHECK_CUDA_CONTIG(*queue_kc);
    TORCH_CHECK(is_bf16(*queue_kc) && queue_kc->size(0) == K &&
                queue_kc->size(1) == C);
    kc = queue_kc->data_ptr();
  }
  at::cuda::CUDAGuard guard(queue.device());
  CHECK_LAUNCH(launch_queue_enqueue(cur_stream(),
                                    queue.data_ptr<float>(), kc,
                                    keys.data_ptr(), is_bf16(keys), C, K, B,
                                    ptr));
}

// ---------------------------------------------------------------------------
void multi_tensor_ema(torch::Tensor pd, torch::Tensor ps, torch::Tensor sizes,
                      double m) {
  CHECK_CUDA_CONTIG(pd);
  CHECK_CUDA_CONTIG(ps);
  CHECK_CUDA_CONTIG(sizes);
  at::cuda::CUDAGuard guard(pd.device());
  CHECK_LAUNCH(launch_multi_tensor_ema(
      cur_stream(), pd.data_ptr<int64_t>(), ps.data_ptr<int64_t>(),
      sizes.data_ptr<int32_t>(), pd.size(0), (float)m));
}

void multi_cast_bf16(torch::Tensor src_ptrs, torch::Tensor dst_ptrs,
                     torch::Tensor sizes) {
  CHECK_CUDA_CONTIG(src_ptrs);
  CHECK_CUDA_CONTIG(dst_ptrs);
  CHECK_CUDA_CONTIG(sizes);
  at::cuda::CUDAGuard guard(src_ptrs.device());
  CHECK_LAUNCH(launch_multi_cast_bf16(
      cur_stream(), src_ptrs.data_ptr<int64_t>(),
      dst_ptrs.data_ptr<int64_t>(), sizes.data_ptr<int32_t>(),
      src_ptrs.size(0)));
}

void multi_transpose_bf16(torch::Tensor src_ptrs, torch::Tensor dst_ptrs,
                          torch::Tensor meta) {
  CHECK_CUDA_CONTIG(src_ptrs);
  CHECK_CUDA_CONTIG(dst_ptrs);
  CHECK_CUDA_CONTIG(meta);
  TORCH_CHECK(meta.numel() == src_ptrs.size(0) * 4);
  at::cuda::CUDAGuard guard(src_ptrs.device());
  CHECK_LAUNCH(launch_multi_transpose_bf16(
      cur_stream(), src_ptrs.data_ptr<int64_t>(),
      dst_ptrs.data_ptr<int64_t>(), meta.data_ptr<int32_t>(),
      src_ptrs.size(0)));
}

void multi_tensor_sgd(torch::Tensor pp, torch::Tensor pg, torch::Tensor pb,
                      torch::Tensor sizes, double lr, double momentum,
                      double wd) {
  at::cuda::CUDAGuard guard(pp.device());
  CHECK_LAUNCH(launch_multi_tensor_sgd(
      cur_stream(), pp.data_ptr<int64_t>(), pg.data_ptr<int64_t>(),
      pb.data_ptr<int64_t>(), sizes.data_ptr<int32_t>(), pp.size(0),
      (float)lr, (float)momentum, (float)wd));
}

void ema_flat(torch::Tensor dst, torch::Tensor src, double m) {
  CHECK_CUDA_CONTIG(dst);
  CHECK_CUDA_CONTIG(src);
  TORCH_CHECK(dst.scalar_type() == torch::kFloat32 &&
              src.scalar_type() == torch::kFloat32 &&
              dst.numel() == src.numel());
  at::cuda::CUDAGuard guard(dst.device());
  CHECK_LAUNCH(launch_ema_flat(cur_stream(), dst.data_ptr<float>(),
                               src.data_ptr<float>(), dst.numel(),
                               (float)m));
}

// ---------------------------------------------------------------------------
// AdamW and the gradient norm over lists of tensors (adamw.hip)

using TensorList = std::vector<torch::Tensor>;

// What these entry points launch goes past the dispatcher, so a tracer would
// take their outputs for constants; FakeTensorMode, make_fx and what is built
// on them run through here with tensors of which there is only the shape.
void check_not_traced(const char* name) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() &&
          !Modes::get_mode(Key::FAKE).has_value() &&
          !Modes::get_mode(Key::PROXY).has_value() &&
          !Modes::get_mode(Key::FUNCTIONAL).has_value(),
      name, " cannot be traced on the GPU");
}

// A subclass that answers for itself when operators are called has no memory
// of its own, and its data pointer may be null.
void check_own_memory(const torch::Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python),
      "a tensor subclass with its own dispatch has no memory for a kernel");
}

// The tensors of a Python list, borrowed: its items hold them during the
// call (owning copies of 800 tensors cost as much time as all checks).
struct Refs {
  std::vector<const torch::Tensor*> t;
  py::object hold;
  Refs() = default;
  explicit Refs(const py::object& list)
      : hold(py::reinterpret_steal<py::object>(PySequence_Fast(
            list.ptr(), "a list of tensors is expected"))) {
    if (!hold) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(hold.ptr());
    t.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* x = PySequence_Fast_GET_ITEM(hold.ptr(), i);
      TORCH_CHECK_TYPE(THPVariable_Check(x), "a list of tensors is expected");
      t.push_back(&THPVariable_Unpack(x));
      check_own_memory(*t.back());
    }
  }
  size_t size() const { return t.size(); }
  bool empty() const { return t.empty(); }
  const torch::Tensor& operator[](size_t i) const { return *t[i]; }
};

int adamw_dtype(const torch::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kHalf: return 2;
    default: break;
  }
  TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, got ",
                   t.scalar_type());
}

// whether a tensor's memory holds its values: not so where it is lazily negated
// (the imaginary part of a conjugate), or a zero that has no memory
bool in_memory(const torch::Tensor& t) {
  return !t.is_neg() && !t._is_zerotensor();
}

// the values, without gaps
torch::Tensor laid_out(const torch::Tensor& t) {
  return in_memory(t) ? t.contiguous()
                      : t.clone(at::MemoryFormat::Contiguous);
}

// same shape and same place of every element (strides of length-1 dims say
// nothing), without gaps
bool same_dense_layout(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  if (!a.is_non_overlapping_and_dense() || !b.is_non_overlapping_and_dense())
    return false;
  if (a.strides() == b.strides()) return true;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// [begin, end) in memory that a launch writes or reads
struct Range {
  uintptr_t begin, end;
  bool write;
};

void add_range(std::vector<Range>& r, const torch::Tensor& t, bool write) {
  if (t.numel() == 0) return;
  const uintptr_t a = (uintptr_t)t.const_data_ptr();
  r.push_back({a, a + t.numel() * t.element_size(), write});
}

// What one workgroup writes no other may touch: a tensor given twice, or two
// views of the same memory, would be a race.
void check_disjoint(std::vector<Range>& r) {
  std::sort(r.begin(), r.end(),
            [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t wrote = 0, read = 0;
  for (const auto& x : r) {
    TORCH_CHECK_VALUE(x.begin >= wrote && !(x.write && x.begin < read),
                      "the tensors of one call must not share memory");
    (x.write ? wrote : read) = std::max(x.write ? wrote : read, x.end);
  }
}

// chunks of n elements, and how many the last one has
int64_t chunks_of(int64_t n, uint16_t& tail) {
  const int64_t chunks = (n + ADAMW_CHUNK - 1) / ADAMW_CHUNK;
  tail = (uint16_t)(n - (chunks - 1) * ADAMW_CHUNK);
  return chunks;
}

// a grid holds fewer than 2^32 threads, 256 of them a chunk
constexpr int64_t MOST_CHUNKS = ((int64_t)1 << 24) - 1;

// 256 MB behind all L2s.  What a call reads and writes may still be there at
// its next use if it fits, and is better kept out of it (and of L2) where it
// does not: ResNet-50's step 183 us through the caches and 147 past them, 2e8
// bf16 weights 818 and 803, the projection head alone (125 MB) 20 and 23.
constexpr int64_t LAST_LEVEL_CACHE = (int64_t)256 << 20;

// room for a tensor in a table; hands the table to `launch` first if needed
template <typename Table, typename F>
int next_slot(Table& tab, int most, int64_t chunks, const F& launch) {
  TORCH_CHECK_VALUE(chunks <= MOST_CHUNKS, "a tensor of over ",
                    MOST_CHUNKS * ADAMW_CHUNK, " elements is too large");
  if (tab.count == most || tab.chunks + chunks > MOST_CHUNKS) {
    launch(tab);
    tab.count = 0, tab.chunks = 0;
  }
  tab.first[tab.count] = tab.chunks;
  tab.chunks += (uint32_t)chunks;
  return tab.count++;
}

// fills AdamwTables of one dtype and hands each to `launch`
template <typename F>
struct TableFiller {
  AdamwTable tab;
  F launch;
  explicit TableFiller(F f) : launch(f) {
    tab.count = 0, tab.chunks = 0, tab.list_base = 0;
  }
  void add(void* p, const void* g, void* m, void* v, void* s, int64_t n,
           size_t number) {
    if ((number >> 16 << 16) != tab.list_base) {
      flush();
      tab.list_base = (uint32_t)(number >> 16 << 16);
    }
    uint16_t tail;
    const int64_t chunks = chunks_of(n, tail);
    const int i = next_slot(tab, ADAMW_TENSORS, chunks, launch);
    tab.p[i] = p, tab.g[i] = g, tab.m[i] = m, tab.v[i] = v, tab.s[i] = s;
    tab.tail[i] = tail, tab.number[i] = (uint16_t)number;
  }
  void flush() {
    if (tab.count) launch(tab);
    tab.count = 0, tab.chunks = 0;
  }
};

// 2-norm over all elements of a list; every tensor dense, on one device.
// again: a step reads the gradients next, so they pass through the caches
// however many they are (2e8 bf16 weights, clipped: 598 us with the norm's
// reads cached, 612 past the caches; 300 MB with nothing after it: 58 and 54)
torch::Tensor grad_norm_checked(const Refs& grads, bool again) {
  auto opts = grads[0].options().dtype(torch::kFloat32).layout(torch::kStrided);
  auto out = torch::empty({}, opts);
  int64_t chunks_in_all = 0, bytes = 0;
  int types = 0;  // a bit for each
  uint16_t tail;
  for (const auto* g : grads.t) {
    if (!g->numel()) continue;
    chunks_in_all += chunks_of(g->numel(), tail);
    bytes += g->nbytes();
    types |= 1 << adamw_dtype(*g, "gradients");
  }
  auto add = [&tail](GradTable& tab, const torch::Tensor& g, const auto& go) {
    const int64_t chunks = chunks_of(g.numel(), tail);
    const int i = next_slot(tab, GRAD_TENSORS, chunks, go);
    tab.g[i] = g.const_data_ptr(), tab.tail[i] = tail;
  };
  if (chunks_in_all <= NORM_SMALL_CHUNKS && (types & (types - 1)) == 0) {
    GradTable tab;
    tab.count = 0, tab.chunks = 0;
    for (const auto* g : grads.t)
      if (g->numel()) add(tab, *g, [](const GradTable&) {});
    CHECK_LAUNCH(launch_norm_small(cur_stream(), &tab, types / 2,
                                   out.data_ptr<float>()));
    return out;
  }
  // workgroups of a launch at most: 8 per CU, which fill it with loads
  constexpr int64_t BLOCKS = 2048;
  const bool once = !again && bytes > LAST_LEVEL_CACHE;
  // a launch takes GRAD_TENSORS tensors of one dtype or MOST_CHUNKS chunks
  const int64_t launches = (int64_t)grads.size() / GRAD_TENSORS + 3 +
                           2 * chunks_in_all / MOST_CHUNKS;
  auto partial = torch::empty({launches * BLOCKS},
                              opts.dtype(torch::kFloat64));
  double* at = partial.data_ptr<double>();
  int64_t used = 0;
  for (int dtype = 0; dtype < 3; ++dtype) {
    if (!(types >> dtype & 1)) continue;
    auto go = [&](const GradTable& tab) {
      // as many as give each the same number of chunks
      const int64_t each = (tab.chunks + BLOCKS - 1) / BLOCKS;
      const int blocks = (int)((tab.chunks + each - 1) / each);
      TORCH_CHECK(used + blocks <= partial.numel());
      CHECK_LAUNCH(launch_sumsq(cur_stream(), &tab, dtype, at + used, blocks,
                                once));
      used += blocks;
    };
    GradTable tab;
    tab.count = 0, tab.chunks = 0;
    for (const auto* g : grads.t)
      if (g->numel() && adamw_dtype(*g, "gradients") == dtype)
        add(tab, *g, go);
    if (tab.count) go(tab);
  }
  CHECK_LAUNCH(launch_norm_final(cur_stream(), at, (int)used,
                                 out.data_ptr<float>()));
  return out;
}

torch::Tensor grad_norm(const py::object& list, bool again) {
  check_not_traced("grad_norm");
  Refs grads(list);
  TORCH_CHECK_VALUE(!grads.empty(), "grad_norm needs at least one tensor");
  const auto device = grads[0].device();
  TORCH_CHECK_VALUE(device.is_cuda(), "gradients must be on one device");
  at::cuda::CUDAGuard guard(device);
  TensorList copies;
  copies.reserve(grads.size());  // their addresses are taken
  for (auto& g : grads.t) {
    TORCH_CHECK_VALUE(g->device() == device,
                      "gradients must be on one device");
    TORCH_CHECK_VALUE(g->layout() == torch::kStrided,
                      "sparse gradients are not supported");
    adamw_dtype(*g, "gradients");
    // an expanded or gapped view is laid out first: each element counts once
    // per place that it has in the tensor
    if (g->is_non_overlapping_and_dense() && in_memory(*g)) continue;
    copies.push_back(laid_out(*g));
    g = &copies.back();
  }
  return grad_norm_checked(grads, again);
}

// One AdamW step (8-bit moments where `scales` is not empty).  Returns the
// gradient norm that the clip went by, if there was one.
c10::optional<torch::Tensor> adamw_step(
    const py::object& params_, const py::object& grads_, const py::object& ms_,
    const py::object& vs_, const py::object& scales_, int64_t step,
    double lr, double beta1, double beta2, double eps, double weight_decay,
    c10::optional<double> max_norm, c10::optional<torch::Tensor> total_norm,
    int64_t seed) {
  const bool eight = !scales_.is_none();
  check_not_traced(eight ? "adamw8bit_" : "adamw_");
  if (total_norm.has_value()) check_own_memory(*total_norm);
  const Refs params(params_), grads(grads_), ms(ms_), vs(vs_);
  const Refs scales = eight ? Refs(scales_) : Refs();
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && ms.size() == n && vs.size() == n &&
                        scales.size() == (eight ? n : 0),
                    "the lists of tensors differ in length");
  if (n == 0) return total_norm;
  const auto device = params[0].device();
  TORCH_CHECK_VALUE(device.is_cuda(), "all tensors must be on one device");
  at::cuda::CUDAGuard guard(device);
  std::vector<Range> ranges;
  ranges.reserve(5 * n);
  const auto m_type = eight ? torch::kFloat8_e4m3fn : torch::kFloat32;
  const auto v_type = eight ? torch::kUInt8 : torch::kFloat32;
  bool seen[3] = {false, false, false};
  for (size_t i = 0; i < n; ++i) {
    const auto &p = params[i], &g = grads[i], &m = ms[i], &v = vs[i];
    seen[adamw_dtype(p, "params")] = true;
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "gradient ", i,
                     " is ", g.scalar_type(), ", its parameter ",
                     p.scalar_type());
    TORCH_CHECK_VALUE(g.layout() == torch::kStrided,
                      "sparse gradients are not supported");
    TORCH_CHECK_TYPE(m.scalar_type() == m_type && v.scalar_type() == v_type,
                     "the moments must be ", m_type, " and ", v_type);
    TORCH_CHECK_VALUE(p.device() == device && g.device() == device &&
                          m.device() == device && v.device() == device,
                      "all tensors must be on one device");
    TORCH_CHECK_VALUE(same_dense_layout(p, g) && same_dense_layout(p, m) &&
                          same_dense_layout(p, v),
                      "parameter ", i, ", its gradient and its moments must "
                      "be dense and laid out alike");
    TORCH_CHECK_VALUE(in_memory(p) && in_memory(g) && in_memory(m) &&
                          in_memory(v) && (!eight || in_memory(scales[i])),
                      "a tensor of parameter ", i, " is lazily negated or a "
                      "zero without memory");
    add_range(ranges, p, true);
    add_range(ranges, g, false);
    add_range(ranges, m, true);
    add_range(ranges, v, true);
    if (eight) {
      const auto& s = scales[i];
      TORCH_CHECK_VALUE(
          s.device() == device && s.scalar_type() == torch::kFloat32 &&
              s.is_contiguous() && s.dim() == 2 &&
              s.size(0) == (p.numel() + 255) / 256 && s.size(1) == 2,
          "scales of parameter ", i, " must be contiguous float32 [",
          (p.numel() + 255) / 256, ", 2]");
      TORCH_CHECK_VALUE((uintptr_t)s.const_data_ptr() % 8 == 0,
                        "scales must be aligned to 8 bytes");
      add_range(ranges, s, true);
    }
  }
  int64_t bytes = 0;
  for (const auto& r : ranges) bytes += r.end - r.begin;
  const bool once = bytes > LAST_LEVEL_CACHE;
  if (max_norm.has_value() && total_norm.has_value()) {
    TORCH_CHECK_VALUE(total_norm->device() == device &&
                          total_norm->numel() == 1 && in_memory(*total_norm) &&
                          total_norm->scalar_type() == torch::kFloat32,
                      "total_norm must be one float32 on the tensors' device");
    add_range(ranges, *total_norm, false);
  }
  check_disjoint(ranges);
  const float* norm = nullptr;
  if (max_norm.has_value()) {
    if (!total_norm.has_value()) total_norm = grad_norm_checked(grads, true);
    norm = total_norm->const_data_ptr<float>();
  }
  AdamwScalars h;
  h.beta1 = (float)beta1;
  h.one_minus_beta1 = (float)(1.0 - beta1);
  h.beta2 = (float)beta2;
  h.one_minus_beta2 = (float)(1.0 - beta2);
  h.inv_root_bc2 =
      (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  h.eps = (float)eps;
  h.decay = (float)(1.0 - lr * weight_decay);
  h.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  h.max_norm = (float)max_norm.value_or(0.0);
  const uint32_t key =
      (uint32_t)seed * 0x6A09E667u + (uint32_t)step * 0xA54FF53Au;
  for (int dtype = 0; dtype < 3; ++dtype) {
    if (!seen[dtype]) continue;
    auto go = [&](const AdamwTable& tab) {
      if (eight)
        CHECK_LAUNCH(launch_adamw8(cur_stream(), &tab, &h, norm, dtype,
                                   once, key));
      else
        CHECK_LAUNCH(launch_adamw(cur_stream(), &tab, &h, norm, dtype, once));
    };
    TableFiller<decltype(go)> fill(go);
    for (size_t i = 0; i < n; ++i)
      if (params[i].numel() && adamw_dtype(params[i], "params") == dtype)
        fill.add(params[i].data_ptr(), grads[i].const_data_ptr(),
                 ms[i].data_ptr(), vs[i].data_ptr(),
                 eight ? scales[i].data_ptr() : nullptr, params[i].numel(),
                 i);
    fill.flush();
  }
  // autograd's count of writes: a graph that saved a weight notices
  for (const Refs* list : {&params, &ms, &vs, &scales})
    for (const auto* t : list->t)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return total_norm;
}

// decoded moments of 8-bit codes
std::pair<TensorList, TensorList> adamw8bit_values(const py::object& ms_,
                                                   const py::object& vs_,
                                                   const py::object& scales_,
                                                   const py::object& dtype_) {
  check_not_traced("adamw8bit_values");
  const Refs ms(ms_), vs(vs_), scales(scales_);
  const auto dtype = torch::python::detail::py_object_to_dtype(dtype_);
  TORCH_CHECK_VALUE(vs.size() == ms.size() && scales.size() == ms.size(),
                    "the lists of tensors differ in length");
  std::pair<TensorList, TensorList> out;
  if (ms.empty()) return out;
  TORCH_CHECK_VALUE(ms[0].is_cuda(), "all tensors must be on one device");
  at::cuda::CUDAGuard guard(ms[0].device());
  int kind = 0;
  auto go = [&](const AdamwTable& tab) {
    CHECK_LAUNCH(launch_adamw8_values(cur_stream(), &tab, kind));
  };
  TableFiller<decltype(go)> fill(go);
  for (size_t i = 0; i < ms.size(); ++i) {
    const auto &m = ms[i], &v = vs[i], &s = scales[i];
    TORCH_CHECK_TYPE(m.scalar_type() == torch::kFloat8_e4m3fn &&
                         v.scalar_type() == torch::kUInt8,
                     "the codes must be float8_e4m3fn and uint8");
    TORCH_CHECK_VALUE(m.device() == ms[0].device() &&
                          v.device() == ms[0].device() &&
                          s.device() == ms[0].device(),
                      "all tensors must be on one device");
    TORCH_CHECK_VALUE(same_dense_layout(m, v),
                      "codes ", i, " must be dense and laid out alike");
    TORCH_CHECK_VALUE(in_memory(m) && in_memory(v) && in_memory(s),
                      "codes ", i, " are lazily negated or zeros without "
                      "memory");
    TORCH_CHECK_VALUE(s.scalar_type() == torch::kFloat32 &&
                          s.is_contiguous() && s.dim() == 2 &&
                          s.size(0) == (m.numel() + 255) / 256 &&
                          s.size(1) == 2 &&
                          (uintptr_t)s.const_data_ptr() % 8 == 0,
                      "scales ", i, " must be contiguous float32 [",
                      (m.numel() + 255) / 256, ", 2], aligned to 8 bytes");
    auto om = torch::empty_strided(m.sizes(), m.strides(),
                                   m.options().dtype(dtype));
    auto ov = torch::empty_strided(m.sizes(), m.strides(),
                                   m.options().dtype(dtype));
    kind = adamw_dtype(om, "values");
    if (m.numel())
      fill.add(om.data_ptr(), ov.data_ptr(), m.data_ptr(), v.data_ptr(),
               s.data_ptr(), m.numel(), 0);
    out.first.push_back(om);
    out.second.push_back(ov);
  }
  fill.flush();
  return out;
}

// ---------------------------------------------------------------------------
// Norms after and before a residual block (norm_residual.hip)

using OptTensor = c10::optional<torch::Tensor>;

// A tensor whose rows (all but the last dimension) lie at equal distances,
// each without gaps: the tensor itself, or a contiguous copy of it.
struct Rows {
  torch::Tensor t;
  int64_t ld = 0;
  Rows() = default;
  explicit Rows(const torch::Tensor& in) : t(in) {
    const int64_t width = in.size(-1);
    ld = width;
    bool ok = (width <= 1 || in.stride(-1) == 1) && in_memory(in);
    int64_t want = -1;  // stride that the next dimension outwards must have
    for (int64_t d = in.dim() - 2; ok && d >= 0; --d) {
      if (in.size(d) == 1) continue;
      if (want < 0) ld = in.stride(d);
      else ok = in.stride(d) == want;
      want = in.stride(d) * in.size(d);
    }
    if (!ok) {
      t = laid_out(in);
      ld = width;
    }
  }
};

struct NormCall {
  NormArgs a{};
  Rows x, h, gate;
  std::vector<torch::Tensor> keep;  // vectors, made contiguous

  const void* vec(const OptTensor& v, int bit) {
    if (!v.has_value()) return nullptr;
    TORCH_CHECK_VALUE(v->is_cuda() && v->device() == x.t.device() &&
                          v->dim() == 1 && v->size(0) == a.width,
                      "a weight, bias or scale must be [", a.width,
                      "] on the device of x");
    const int type = adamw_dtype(*v, "weights, biases and scale");
    TORCH_CHECK_TYPE(type == 0 || type == a.type_h, "weights, biases and "
                     "scale must be float32 or of the block's type, got ",
                     v->scalar_type());
    if (type == 0) a.f32 |= 1 << bit;
    keep.push_back(laid_out(*v));
    return keep.back().const_data_ptr();
  }

  NormCall(const torch::Tensor& x_in, const OptTensor& h_in,
           const OptTensor& gate_in, const OptTensor& w1, const OptTensor& b1,
           const OptTensor& w2, const OptTensor& b2, const OptTensor& scale,
           double scale_value, int64_t post, int64_t pre, int64_t act,
           double post_eps, double pre_eps, int type_y) {
    TORCH_CHECK_VALUE(x_in.is_cuda() && x_in.dim() >= 1 && x_in.size(-1) > 0,
                      "x must be a GPU tensor [..., width]");
    TORCH_CHECK_VALUE(x_in.size(-1) <= NORM_MAX_WIDTH, "a width of ",
                      x_in.size(-1), " is over ", NORM_MAX_WIDTH);
    x = Rows(x_in);
    a.width = (int)x_in.size(-1);
    a.rows = x_in.numel() / a.width;
    a.type_x = adamw_dtype(x_in, "x");
    a.type_h = type_y;
    a.x = x.t.const_data_ptr(), a.ld_x = x.ld;
    if (h_in.has_value()) {
      TORCH_CHECK_VALUE(h_in->sizes() == x_in.sizes() &&
                            h_in->device() == x_in.device(),
                        "branch must have x's shape and device");
      a.type_h = adamw_dtype(*h_in, "branch");
      h = Rows(*h_in);
      a.h = h.t.const_data_ptr(), a.ld_h = h.ld;
    }
    TORCH_CHECK_TYPE(a.type_x == 0 || a.type_x == a.type_h,
                     "x must be float32 or of the block's type");
    if (gate_in.has_value()) {
      const auto& g = *gate_in;
      TORCH_CHECK_VALUE(h_in.has_value() && g.device() == x_in.device() &&
                            g.dim() == x_in.dim() &&
                            g.sizes().slice(0, g.dim() - 1) ==
                                x_in.sizes().slice(0, x_in.dim() - 1) &&
                            (g.size(-1) == a.width || g.size(-1) == 1),
                        "gate must have the branch's shape, or 1 as its last "
                        "dimension");
      TORCH_CHECK_TYPE(adamw_dtype(g, "gate") == a.type_h,
                       "gate must be of the branch's type");
      a.gate_kind = g.size(-1) == a.width ? NORM_GATE_FULL : NORM_GATE_ROW;
      gate = Rows(g);
      a.gate = gate.t.const_data_ptr(), a.ld_g = gate.ld;
    }
    TORCH_CHECK_VALUE(post >= 0 && post <= 2 && pre >= 0 && pre <= 2 &&
                      act >= 0 && act <= 2, "unknown norm or gate");
    a.post = (int)post, a.pre = (int)pre, a.act = (int)act;
    a.scale_value = (float)scale_value;
    a.post_eps = (float)post_eps, a.pre_eps = (float)pre_eps;
    a.w1 = vec(w1, 0), a.b1 = vec(b1, 1), a.w2 = vec(w2, 2);
    a.b2 = vec(b2, 3), a.scale = vec(scale, 4);
  }
};

// straight to the allocator: the dispatcher's part of torch::empty is half of
// its 1.5 us, and a backward pass makes up to nine
torch::Tensor new_tensor(torch::IntArrayRef sizes, torch::ScalarType dtype,
                         const torch::Device& device) {
  return torch::Tensor(
      at::detail::empty_cuda(sizes, dtype, device, c10::nullopt));
}

torch::ScalarType norm_type(int t) {
  return t == 0 ? torch::kFloat32 : t == 1 ? torch::kBFloat16 : torch::kHalf;
}

// what is not a tensor of a call
struct NormNumbers {
  double scale_value, post_eps, pre_eps;
  int64_t post, pre, act, type_y;
};

// {r, y, stats}; undefined where there is none
std::array<torch::Tensor, 3> norm_residual_fwd(
    const torch::Tensor& x, const OptTensor& h, const OptTensor& gate,
    const OptTensor& w1, const OptTensor& b1, const OptTensor& w2,
    const OptTensor& b2, const OptTensor& scale, const NormNumbers& num,
    bool want_stats) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a GPU tensor");
  at::cuda::CUDAGuard guard(x.device());
  at::NoGradGuard no_grad;  // copies of strided inputs need no graph
  NormCall c(x, h, gate, w1, b1, w2, b2, scale, num.scale_value, num.post,
             num.pre, num.act, num.post_eps, num.pre_eps, (int)num.type_y);
  std::array<torch::Tensor, 3> out;
  if (h.has_value()) {
    out[0] = new_tensor(x.sizes(), x.scalar_type(), x.device());
    c.a.r = out[0].data_ptr();
  }
  if (num.pre != NORM_NONE) {
    out[1] = new_tensor(x.sizes(), norm_type(c.a.type_h), x.device());
    c.a.y = out[1].data_ptr();
  }
  if (want_stats) {
    out[2] = new_tensor({4, c.a.rows}, torch::kFloat32, x.device());
    c.a.stats = out[2].data_ptr<float>();
  }
  CHECK_LAUNCH(launch_norm_fwd(cur_stream(), &c.a));
  return out;
}

// {dx, dh, dgate, dw1, db1, dw2, db2, dscale}, those that `want` has a bit
// for
std::vector<torch::Tensor> norm_residual_bwd(
    const OptTensor& d_r, const OptTensor& d_y, const torch::Tensor& stats,
    const torch::Tensor& x, const OptTensor& h, const OptTensor& gate,
    const OptTensor& w1, const OptTensor& b1, const OptTensor& w2,
    const OptTensor& b2, const OptTensor& scale, const NormNumbers& num,
    int64_t want) {
  at::cuda::CUDAGuard guard(x.device());
  NormCall c(x, h, gate, w1, b1, w2, b2, scale, num.scale_value, num.post,
             num.pre, num.act, num.post_eps, num.pre_eps, (int)num.type_y);
  TORCH_CHECK(stats.is_cuda() && stats.is_contiguous() &&
              stats.scalar_type() == torch::kFloat32 &&
              stats.numel() == 4 * c.a.rows);
  c.a.stats = stats.data_ptr<float>();
  NormGrads o{};
  const auto type_h = norm_type(c.a.type_h);
  torch::Tensor dr, dy;
  if (d_r.has_value()) {
    TORCH_CHECK(d_r->sizes() == x.sizes() &&
                d_r->scalar_type() == x.scalar_type() &&
                d_r->device() == x.device());
    dr = laid_out(*d_r);
    o.d_r = dr.const_data_ptr();
  }
  if (d_y.has_value()) {
    TORCH_CHECK(d_y->sizes() == x.sizes() && d_y->scalar_type() == type_h &&
                d_y->device() == x.device() && num.pre != NORM_NONE);
    dy = laid_out(*d_y);
    o.d_y = dy.const_data_ptr();
  }
  std::vector<torch::Tensor> out(8);
  if (want & 1) {
    out[0] = new_tensor(x.sizes(), x.scalar_type(), x.device());
    o.d_x = out[0].data_ptr();
  }
  if ((want & 2) && h.has_value()) {
    out[1] = new_tensor(x.sizes(), type_h, x.device());
    o.d_h = out[1].data_ptr();
  }
  if ((want & 4) && gate.has_value()) {
    out[2] = new_tensor(gate->sizes(), type_h, x.device());
    o.d_gate = out[2].data_ptr();
  }
  const OptTensor* vec[5] = {&w1, &b1, &w2, &b2, &scale};
  void** d_vec[5] = {&o.d_w1, &o.d_b1, &o.d_w2, &o.d_b2, &o.d_scale};
  for (int j = 0; j < 5; ++j) {
    if (!((want >> (3 + j)) & 1) || !vec[j]->has_value()) continue;
    auto& d = out[3 + j];
    d = new_tensor({c.a.width}, (*vec[j])->scalar_type(), x.device());
    *d_vec[j] = d.data_ptr();
    // no rows: nothing is launched, and the sums are zero
    if (!c.a.rows) d.zero_();
  }
  if (!c.a.rows) return out;
  const bool sums[4] = {o.d_w1 || o.d_scale,
                        o.d_b1 || (o.d_scale && c.a.b1), o.d_w2 != nullptr,
                        o.d_b2 != nullptr};
  const int n = sums[0] + sums[1] + sums[2] + sums[3];
  const int blocks = norm_bwd_blocks(&c.a);
  const int64_t slab = (int64_t)blocks * c.a.width;
  torch::Tensor partial;
  if (n) {
    partial = new_tensor({n * slab}, torch::kFloat32, x.device());
    float* at = partial.data_ptr<float>();
    for (int j = 0; j < 4; ++j)
      if (sums[j]) o.partial[j] = at, at += slab;
  }
  CHECK_LAUNCH(launch_norm_bwd(cur_stream(), &c.a, &o, blocks));
  if (n) CHECK_LAUNCH(launch_norm_columns(cur_stream(), &c.a, &o, blocks));
  return out;
}

// The autograd node of a call.  (A Node, and not a torch::autograd::Function,
// which wraps every argument and keeps what is no tensor in a dictionary:
// 256 x 2048 both ways takes 105 us against 112.)
struct NormResidualBackward : public torch::autograd::Node {
  // x, branch, gate, post's weight and bias, pre's, scale
  std::array<torch::autograd::SavedVariable, 8> saved;
  torch::Tensor stats;
  NormNumbers num;
  bool has_r = false, has_y = false;

  std::string name() const override { return "NormResidualBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved) s.reset_data();
    stats.reset();
  }

  torch::autograd::variable_list apply(
      torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(stats.defined(), torch::autograd::ERR_BACKWARD_TWICE);
    check_not_traced("norm_residual's backward pass");
    torch::Tensor t[8];
    bool again = false;  // a graph of the backward pass is asked for
    for (int i = 0; i < 8; ++i) {
      t[i] = saved[i].unpack();
      if (!t[i].defined()) continue;
      check_own_memory(t[i]);
      again |= t[i].requires_grad();
    }
    for (const auto& g : grads) {
      if (!g.defined()) continue;
      check_own_memory(g);
      again |= g.requires_grad();
    }
    auto opt = [](const torch::Tensor& v) {
      return v.defined() ? OptTensor(v) : OptTensor();
    };
    size_t at = 0;
    OptTensor d_r, d_y;
    if (has_r) d_r = opt(grads.at(at++));
    if (has_y) d_y = opt(grads.at(at++));
    if (!d_r.has_value() && !d_y.has_value())
      return torch::autograd::variable_list(8);
    int64_t want = 0;
    for (int i = 0; i < 8; ++i)
      if (task_should_compute_output(i)) want |= 1 << i;
    auto out = norm_residual_bwd(d_r, d_y, stats, t[0], opt(t[1]), opt(t[2]),
                                 opt(t[3]), opt(t[4]), opt(t[5]), opt(t[6]),
                                 opt(t[7]), num, want);
    if (again && at::GradMode::is_enabled()) {
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "norm_residual has no second derivatives", (int64_t)out.size());
      out = (*error)(std::move(out));
    }
    return out;
  }
};

// (r or None, y or None), with a backward pass where one may follow
std::pair<OptTensor, OptTensor> norm_residual(
    const torch::Tensor& x, const OptTensor& h, const OptTensor& gate,
    const OptTensor& w1, const OptTensor& b1, const OptTensor& w2,
    const OptTensor& b2, const OptTensor& scale, double scale_value,
    int64_t post, int64_t pre, int64_t act, double post_eps, double pre_eps,
    int64_t type_y) {
  if (const auto& func = at::functorch::functorchTLSAccessor())
    func->checkSupportsCppAutogradFunction();
  check_not_traced("norm_residual");
  check_own_memory(x);
  bool train = x.requires_grad(), tangent = x._fw_grad(0).defined();
  for (auto* t : {&h, &gate, &w1, &b1, &w2, &b2, &scale}) {
    if (!t->has_value()) continue;
    check_own_memory(**t);
    train |= (*t)->requires_grad();
    tangent |= (*t)->_fw_grad(0).defined();
  }
  TORCH_CHECK_NOT_IMPLEMENTED(
      !tangent, "norm_residual has no forward-mode derivatives on the GPU");
  train = train && at::GradMode::is_enabled();
  const NormNumbers num{scale_value, post_eps, pre_eps, post,
                        pre,         act,      type_y};
  auto got = norm_residual_fwd(x, h, gate, w1, b1, w2, b2, scale, num, train);
  if (train) {
    std::shared_ptr<NormResidualBackward> node(new NormResidualBackward(),
                                               torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(
        x, h, gate, w1, b1, w2, b2, scale));
    node->saved[0] = torch::autograd::SavedVariable(x, false);
    int i = 1;
    for (auto* t : {&h, &gate, &w1, &b1, &w2, &b2, &scale})
      node->saved[i++] =
          torch::autograd::SavedVariable(t->value_or(torch::Tensor()), false);
    node->stats = got[2];
    node->num = num;
    node->has_r = got[0].defined();
    node->has_y = got[1].defined();
    for (int k = 0; k < 2; ++k)
      if (got[k].defined()) torch::autograd::set_history(got[k], node);
  }
  std::pair<OptTensor, OptTensor> out;
  if (got[0].defined()) out.first = got[0];
  if (got[1].defined()) out.second = got[1];
  return out;
}

// ---------------------------------------------------------------------------
// Fused BatchNorm (+ReLU, +residual).  x is a channels_last [N,C,H,W] bf16
// tensor viewed here as [R, C] with R = N*H*W.

std::vector<torch::Tensor> bn_fwd_train(torch::Tensor x,
                                        c10::optional<torch::Tensor> res,
                                        torch::Tensor gamma,
                                        torch::Tensor beta,
                                        c10::optional<torch::Tensor> rmean,
                                        c10::optional<torch::Tensor> rvar,
                                        double eps, double momentum,
                                        bool relu) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x));
  const int64_t C = x.size(1);
  const int64_t R = x.numel() / C;
  at::cuda::CUDAGuard guard(x.device());
  auto f32 = x.options().dtype(torch::kFloat32);
  auto part_s = torch::empty({1024, C}, f32);
  auto part_q = torch::empty({1024, C}, f32);
  auto mean = torch::empty({C}, f32);
  auto rstd = torch::empty({C}, f32);
  CHECK_LAUNCH(launch_bn_stats(
      cur_stream(), x.data_ptr(), part_s.data_ptr<float>(),
      part_q.data_ptr<float>(), mean.data_ptr<float>(),
      rstd.data_ptr<float>(),
      rmean.has_value() ? rmean->data_ptr<float>() : nullptr,
      rvar.has_value() ? rvar->data_ptr<float>() : nullptr, R, C, (float)eps,
      (float)momentum));
  auto y = torch::empty_like(x);
  CHECK_LAUNCH(launch_bn_apply(
      cur_stream(), x.data_ptr(),
      res.has_value() ? res->data_ptr() : nullptr, y.data_ptr(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      gamma.data_ptr<float>(), beta.data_ptr<float>(), R, C, relu));
  return {y, mean, rstd};
}

torch::Tensor bn_fwd_eval(torch::Tensor x, c10::optional<torch::Tensor> res,
                          torch::Tensor gamma, torch::Tensor beta,
                          torch::Tensor mean, torch::Tensor rstd, bool relu) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x));
  const int64_t C = x.size(1);
  const int64_t R = x.numel() / C;
  at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty_like(x);
  CHECK_LAUNCH(launch_bn_apply(
      cur_stream(), x.data_ptr(),
      res.has_value() ? res->data_ptr() : nullptr, y.data_ptr(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      gamma.data_ptr<float>(), beta.data_ptr<float>(), R, C, relu));
  return y;
}

std::vector<torch::Tensor> bn_bwd(torch::Tensor g, torch::Tensor y,
                                  torch::Tensor x, torch::Tensor mean,
                                  torch::Tensor rstd, torch::Tensor gamma,
                                  bool relu, bool train, bool need_dres) {
  TORCH_CHECK(g.is_cuda() && is_bf16(g));
  const int64_t C = x.size(1);
  const int64_t R = x.numel() / C;
  at::cuda::CUDAGuard guard(x.device());
  auto f32 = x.options().dtype(torch::kFloat32);
  auto part_db = torch::empty({1024, C}, f32);
  auto part_dg = torch::empty({1024, C}, f32);
  auto dbeta = torch::empty({C}, f32);
  auto dgamma = torch::empty({C}, f32);
  CHECK_LAUNCH(launch_bn_bwd_reduce(
      cur_stream(), g.data_ptr(), y.data_ptr(), x.data_ptr(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      part_db.data_ptr<float>(), part_dg.data_ptr<float>(),
      dbeta.data_ptr<float>(), dgamma.data_ptr<float>(), R, C, relu));
  auto dx = torch::empty_like(g);
  torch::Tensor dres;
  if (need_dres) dres = torch::empty_like(g);
  CHECK_LAUNCH(launch_bn_bwd_dx(
      cur_stream(), g.data_ptr(), y.data_ptr(), x.data_ptr(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      gamma.data_ptr<float>(), dbeta.data_ptr<float>(),
      dgamma.data_ptr<float>(), dx.data_ptr(),
      need_dres ? dres.data_ptr() : nullptr, R, C, relu, train));
  if (need_dres) return {dx, dgamma, dbeta, dres};
  return {dx, dgamma, dbeta};
}

// ---------------------------------------------------------------------------
// bf16 NT-GEMM (1x1-conv forward/dgrad): C[M,N] = A[M,K] @ Bt[N,K]^T.
// c_add (optional): epilogue C += c_add — fuses the residual-path gradient
// accumulation into the dgrad GEMM store tail.
torch::Tensor gemm_nt_bf16(torch::Tensor A, torch::Tensor Bt,
                           c10::optional<torch::Tensor> c_add) {
  CHECK_CUDA_CONTIG(A);
  CHECK_CUDA_CONTIG(Bt);
  TORCH_CHECK(is_bf16(A) && is_bf16(Bt) && A.size(1) == Bt.size(1));
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  if (c_add.has_value())
    TORCH_CHECK(is_bf16(*c_add) && c_add->is_contiguous() &&
                c_add->numel() == M * N);
  at::cuda::CUDAGuard guard(A.device());
  auto C = torch::empty({M, N}, A.options());
  // LDS-staged kernel for conforming shapes, naive fragment-load fallback
  CHECK_LAUNCH(launch_gemm_nt_lds_bf16(
      cur_stream(), A.data_ptr(), Bt.data_ptr(), C.data_ptr(), M, N, K,
      c_add.has_value() ? c_add->data_ptr() : nullptr));
  return C;
}

// GEMM with fused BN-apply (A path) / BN-stats (output) — the conv+BN hot
// path.  want_aout materializes the transformed A operand (consumer conv
// backward wgrad input); c_add fuses an epilogue add.
std::vector<torch::Tensor> gemm_nt_fused(
    torch::Tensor A, torch::Tensor Bt, c10::optional<torch::Tensor> a_scale,
    c10::optional<torch::Tensor> a_shift, bool a_relu, bool want_stats,
    bool want_aout, c10::optional<torch::Tensor> c_add,
    c10::optional<torch::Tensor> ws_sum,
    c10::optional<torch::Tensor> ws_ssq) {
  CHECK_CUDA_CONTIG(A);
  CHECK_CUDA_CONTIG(Bt);
  TORCH_CHECK(is_bf16(A) && is_bf16(Bt) && A.size(1) == Bt.size(1));
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  TORCH_CHECK(a_scale.has_value() == a_shift.has_value());
  if (a_scale.has_value())
    TORCH_CHECK(a_scale->numel() == K && a_shift->numel() == K);
  TORCH_CHECK(!want_aout || a_scale.has_value(),
              "want_aout requires the BN-apply prologue");
  if (c_add.has_value())
    TORCH_CHECK(is_bf16(*c_add) && c_add->is_contiguous() &&
                c_add->numel() == M * N);
  at::cuda::CUDAGuard guard(A.device());
  auto C = torch::empty({M, N}, A.options());
  torch::Tensor ssum, ssq, aout;
  if (want_stats) {
    // slot-striped [256, N] partials (see conv1x1.hip STAT_SLOTS);
    // bn_finalize reduces the slots.  When the caller provides a
    // workspace pair it must be pre-zeroed — the finalize(zero_src=True)
    // restores that invariant, so no fill kernels run per step.
    if (ws_sum.has_value()) {
      TORCH_CHECK(ws_sum->numel() == 256 * N && ws_sum->is_contiguous() &&
                  ws_ssq->numel() == 256 * N && ws_ssq->is_contiguous());
      ssum = *ws_sum;
      ssq = *ws_ssq;
    } else {
      ssum = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
      ssq = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
    }
  }
  if (want_aout) aout = torch::empty({M, K}, A.options());
  CHECK_LAUNCH(launch_gemm_nt_fused_bf16(
      cur_stream(), A.data_ptr(), Bt.data_ptr(), C.data_ptr(), M, N, K,
      a_scale.has_value() ? a_scale->data_ptr<float>() : nullptr,
      a_shift.has_value() ? a_shift->data_ptr<float>() : nullptr, a_relu,
      want_stats ? ssum.data_ptr<float>() : nullptr,
      want_stats ? ssq.data_ptr<float>() : nullptr,
      want_aout ? aout.data_ptr() : nullptr,
      c_add.has_value() ? c_add->data_ptr() : nullptr));
  std::vector<torch::Tensor> out = {C};
  if (want_stats) {
    out.push_back(ssum);
    out.push_back(ssq);
  }
  if (want_aout) out.push_back(aout);
  return out;
}

// fp8 e4m3 GEMM (MX-scaled MFMA, per-tensor software scaling):
// C_bf16 = (A8 @ B8t^T) * out_scale.  want_stats adds the bn-stats
// epilogue ([256, N] slot slabs like the bf16 path).
std::vector<torch::Tensor> gemm_nt_fp8(torch::Tensor A, torch::Tensor Bt,
                                       double out_scale, bool want_stats,
                                       c10::optional<torch::Tensor> ws_sum,
                                       c10::optional<torch::Tensor> ws_ssq) {
  CHECK_CUDA_CONTIG(A);
  CHECK_CUDA_CONTIG(Bt);
  TORCH_CHECK(A.scalar_type() == torch::kFloat8_e4m3fn &&
              Bt.scalar_type() == torch::kFloat8_e4m3fn &&
              A.size(1) == Bt.size(1));
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  at::cuda::CUDAGuard guard(A.device());
  auto C = torch::empty({M, N}, A.options().dtype(torch::kBFloat16));
  torch::Tensor ssum, ssq;
  if (want_stats) {
    if (ws_sum.has_value()) {
      ssum = *ws_sum;
      ssq = *ws_ssq;
    } else {
      ssum = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
      ssq = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
    }
  }
  CHECK_LAUNCH(launch_gemm_nt_fp8(
      cur_stream(), A.data_ptr(), Bt.data_ptr(), C.data_ptr(), M, N, K,
      (float)out_scale, want_stats ? ssum.data_ptr<float>() : nullptr,
      want_stats ? ssq.data_ptr<float>() : nullptr));
  if (want_stats) return {C, ssum, ssq};
  return {C};
}

// ---------------------------------------------------------------------------
// Granular BN entry points for the conv+BN fused block path.

// stats only (1 read): mean/rstd + running-stats update
std::vector<torch::Tensor> bn_stats(torch::Tensor x,
                                    c10::optional<torch::Tensor> rmean,
                                    c10::optional<torch::Tensor> rvar,
                                    double eps, double momentum) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x));
  const int64_t C = x.size(1);
  const int64_t R = x.numel() / C;
  at::cuda::CUDAGuard guard(x.device());
  auto f32 = x.options().dtype(torch::kFloat32);
  auto part_s = torch::empty({1024, C}, f32);
  auto part_q = torch::empty({1024, C}, f32);
  auto mean = torch::empty({C}, f32);
  auto rstd = torch::empty({C}, f32);
  CHECK_LAUNCH(launch_bn_stats(
      cur_stream(), x.data_ptr(), part_s.data_ptr<float>(),
      part_q.data_ptr<float>(), mean.data_ptr<float>(),
      rstd.data_ptr<float>(),
      rmean.has_value() ? rmean->data_ptr<float>() : nullptr,
      rvar.has_value() ? rvar->data_ptr<float>() : nullptr, R, C, (float)eps,
      (float)momentum));
  return {mean, rstd};
}

// finalize from the conv-GEMM epilogue's slot-striped channel partials
// ([P, C]; 1-D input means P = 1)
std::vector<torch::Tensor> bn_finalize(torch::Tensor ssum, torch::Tensor ssq,
                                       int64_t R,
                                       c10::optional<torch::Tensor> rmean,
                                       c10::optional<torch::Tensor> rvar,
                                       double eps, double momentum,
                                       bool zero_src) {
  CHECK_CUDA_CONTIG(ssum);
  CHECK_CUDA_CONTIG(ssq);
  const int64_t C = ssum.dim() == 2 ? ssum.size(1) : ssum.numel();
  const int64_t P = ssum.dim() == 2 ? ssum.size(0) : 1;
  at::cuda::CUDAGuard guard(ssum.device());
  auto mean = torch::empty({C}, ssum.options());
  auto rstd = torch::empty({C}, ssum.options());
  CHECK_LAUNCH(launch_bn_finalize(
      cur_stream(), ssum.data_ptr<float>(), ssq.data_ptr<float>(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      rmean.has_value() ? rmean->data_ptr<float>() : nullptr,
      rvar.has_value() ? rvar->data_ptr<float>() : nullptr, R, C, P,
      (float)eps, (float)momentum, zero_src));
  return {mean, rstd};
}

// dx-only backward: upstream grad already relu-masked (by the dgrad-GEMM
// epilogue), dbeta/dgamma already reduced there — one elementwise pass.
torch::Tensor bn_bwd_dx_only(torch::Tensor gp, torch::Tensor z,
                             torch::Tensor mean, torch::Tensor rstd,
                             torch::Tensor gamma, torch::Tensor dbeta,
                             torch::Tensor dgamma) {
  TORCH_CHECK(gp.is_cuda() && is_bf16(gp) && is_bf16(z));
  const int64_t C = z.size(1);
  const int64_t R = z.numel() / C;
  at::cuda::CUDAGuard guard(z.device());
  auto dx = torch::empty_like(gp);
  CHECK_LAUNCH(launch_bn_bwd_dx(
      cur_stream(), gp.data_ptr(), gp.data_ptr(), z.data_ptr(),
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      gamma.data_ptr<float>(), dbeta.data_ptr<float>(),
      dgamma.data_ptr<float>(), dx.data_ptr(), nullptr, R, C,
      /*relu=*/false, /*train=*/true));
  return dx;
}

// Round-2 prototype: 3x3 pad-1 conv (stride 1/2) as implicit MFMA GEMM,
// with optional fused BN-apply (input path) / BN-stats (output).
std::vector<torch::Tensor> conv3x3_fwd(
    torch::Tensor x, torch::Tensor w, int64_t stride,
    c10::optional<torch::Tensor> a_scale, c10::optional<torch::Tensor> a_shift,
    bool a_relu, bool want_stats, c10::optional<torch::Tensor> neutral) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x) && x.dim() == 4);
  TORCH_CHECK(is_bf16(w) && w.dim() == 4 && w.size(2) == 3 && w.size(3) == 3);
  TORCH_CHECK(x.is_contiguous(torch::MemoryFormat::ChannelsLast) &&
              w.is_contiguous(torch::MemoryFormat::ChannelsLast),
              "conv3x3_fwd wants channels_last x and w");
  const int64_t N = x.size(0), Ci = x.size(1), H = x.size(2), W = x.size(3);
  const int64_t Co = w.size(0);
  TORCH_CHECK(w.size(1) == Ci);
  const int64_t Ho = (H - 1) / stride + 1, Wo = (W - 1) / stride + 1;
  at::cuda::CUDAGuard guard(x.device());
  auto out = torch::empty({N, Co, Ho, Wo}, x.options())
                 .contiguous(torch::MemoryFormat::ChannelsLast);
  torch::Tensor zp;
  if (neutral.has_value()) {
    TORCH_CHECK(is_bf16(*neutral) && neutral->numel() >= Ci + 8);
    zp = *neutral;
  } else {
    zp = torch::zeros({Ci + 8}, x.options());
  }
  torch::Tensor ssum, ssq;
  if (want_stats) {
    ssum = torch::zeros({Co}, x.options().dtype(torch::kFloat32));
    ssq = torch::zeros({Co}, x.options().dtype(torch::kFloat32));
  }
  CHECK_LAUNCH(launch_conv3x3_fwd(
      cur_stream(), x.data_ptr(), w.data_ptr(), zp.data_ptr(),
      out.data_ptr(), N, H, W, Ci, Co, stride,
      a_scale.has_value() ? a_scale->data_ptr<float>() : nullptr,
      a_shift.has_value() ? a_shift->data_ptr<float>() : nullptr, a_relu,
      want_stats ? ssum.data_ptr<float>() : nullptr,
      want_stats ? ssq.data_ptr<float>() : nullptr));
  if (want_stats) return {out, ssum, ssq};
  return {out};
}

torch::Tensor conv1x1_strided(torch::Tensor x, torch::Tensor w,
                              int64_t stride) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x) && x.dim() == 4);
  TORCH_CHECK(is_bf16(w) && w.dim() == 4 && w.size(2) == 1 && w.size(3) == 1);
  TORCH_CHECK(x.is_contiguous(torch::MemoryFormat::ChannelsLast));
  const int64_t N = x.size(0), Ci = x.size(1), H = x.size(2), W = x.size(3);
  const int64_t Co = w.size(0);
  TORCH_CHECK(w.size(1) == Ci);
  const int64_t Ho = (H - 1) / stride + 1, Wo = (W - 1) / stride + 1;
  at::cuda::CUDAGuard guard(x.device());
  auto out = torch::empty({N, Co, Ho, Wo}, x.options())
                 .contiguous(torch::MemoryFormat::ChannelsLast);
  CHECK_LAUNCH(launch_conv1x1_strided(cur_stream(), x.data_ptr(),
                                      w.contiguous().data_ptr(),
                                      out.data_ptr(), N, H, W, Ci, Co,
                                      stride));
  return out;
}

// Round-2 prototype: dgrad GEMM + fused BN-backward epilogue.
std::vector<torch::Tensor> gemm_nt_dgrad_epi(torch::Tensor A,
                                             torch::Tensor Bt,
                                             torch::Tensor y, torch::Tensor z,
                                             torch::Tensor mean,
                                             torch::Tensor rstd,
                                             c10::optional<torch::Tensor>
                                                 c_add,
                                             c10::optional<torch::Tensor>
                                                 ws_db,
                                             c10::optional<torch::Tensor>
                                                 ws_dg) {
  CHECK_CUDA_CONTIG(A);
  CHECK_CUDA_CONTIG(Bt);
  TORCH_CHECK(is_bf16(A) && is_bf16(Bt) && is_bf16(y) && is_bf16(z));
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  TORCH_CHECK(y.numel() == M * N && z.numel() == M * N);
  TORCH_CHECK(mean.numel() == N && rstd.numel() == N);
  if (c_add.has_value())
    TORCH_CHECK(is_bf16(*c_add) && c_add->is_contiguous() &&
                c_add->numel() == M * N);
  at::cuda::CUDAGuard guard(A.device());
  auto C = torch::empty({M, N}, A.options());
  // slot-striped partials (conv1x1.hip STAT_SLOTS), reduced by the
  // self-zeroing slot_reduce2 (caller workspace must be pre-zeroed)
  torch::Tensor dbeta, dgamma;
  if (ws_db.has_value()) {
    TORCH_CHECK(ws_db->numel() == 256 * N && ws_db->is_contiguous() &&
                ws_dg->numel() == 256 * N && ws_dg->is_contiguous());
    dbeta = *ws_db;
    dgamma = *ws_dg;
  } else {
    dbeta = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
    dgamma = torch::zeros({256, N}, A.options().dtype(torch::kFloat32));
  }
  CHECK_LAUNCH(launch_gemm_nt_dgrad_epi(
      cur_stream(), A.data_ptr(), Bt.data_ptr(), C.data_ptr(), M, N, K,
      y.data_ptr(), z.data_ptr(), mean.data_ptr<float>(),
      rstd.data_ptr<float>(), dbeta.data_ptr<float>(),
      dgamma.data_ptr<float>(),
      c_add.has_value() ? c_add->data_ptr() : nullptr));
  auto db = torch::empty({N}, A.options().dtype(torch::kFloat32));
  auto dg = torch::empty({N}, A.options().dtype(torch::kFloat32));
  CHECK_LAUNCH(launch_slot_reduce2(
      cur_stream(), dbeta.data_ptr<float>(), dgamma.data_ptr<float>(),
      db.data_ptr<float>(), dg.data_ptr<float>(), N, 256));
  return {C, db, dg};
}

// ---------------------------------------------------------------------------
// MaxPool2d 3x3/s2/p1 (ResNet stem), NHWC bf16
std::vector<torch::Tensor> maxpool_fwd(torch::Tensor x) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x) && x.dim() == 4);
  const int64_t N = x.size(0), C = x.size(1), H = x.size(2), W = x.size(3);
  const int64_t Ho = (H + 1) / 2, Wo = (W + 1) / 2;
  at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty({N, C, Ho, Wo}, x.options())
               .contiguous(torch::MemoryFormat::ChannelsLast);
  auto idx = torch::empty({N, Ho, Wo, C}, x.options().dtype(torch::kUInt8));
  CHECK_LAUNCH(launch_maxpool_fwd(cur_stream(), x.data_ptr(), y.data_ptr(),
                                  idx.data_ptr(), N, C, H, W, Ho, Wo));
  return {y, idx};
}

// head adaptive-avg-pool to 1x1 (NHWC bf16)
torch::Tensor avgpool_fwd(torch::Tensor x) {
  TORCH_CHECK(x.is_cuda() && is_bf16(x) && x.dim() == 4);
  const int64_t N = x.size(0), C = x.size(1), H = x.size(2), W = x.size(3);
  at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty({N, C, 1, 1}, x.options())
               .contiguous(torch::MemoryFormat::ChannelsLast);
  CHECK_LAUNCH(launch_avgpool_fwd(cur_stream(), x.data_ptr(), y.data_ptr(),
                                  N, C, H * W));
  return y;
}

torch::Tensor avgpool_bwd(torch::Tensor g, int64_t H, int64_t W) {
  TORCH_CHECK(g.is_cuda() && is_bf16(g));
  const int64_t N = g.size(0), C = g.size(1);
  at::cuda::CUDAGuard guard(g.device());
  auto dx = torch::empty({N, C, H, W}, g.options())
                .contiguous(torch::MemoryFormat::ChannelsLast);
  CHECK_LAUNCH(launch_avgpool_bwd(cur_stream(), g.data_ptr(), dx.data_ptr(),
                                  N, C, H * W));
  return dx;
}

torch::Tensor maxpool_bwd(torch::Tensor g, torch::Tensor idx, int64_t H,
                          int64_t W) {
  TORCH_CHECK(g.is_cuda() && is_bf16(g) && g.dim() == 4);
  const int64_t N = g.size(0), C = g.size(1), Ho = g.size(2), Wo = g.size(3);
  at::cuda::CUDAGuard guard(g.device());
  auto dx = torch::empty({N, C, H, W}, g.options())
                .contiguous(torch::MemoryFormat::ChannelsLast);
  CHECK_LAUNCH(launch_maxpool_bwd(cur_stream(), g.data_ptr(), idx.data_ptr(),
                                  dx.data_ptr(), N, C, H, W, Ho, Wo));
  return dx;
}

// ---------------------------------------------------------------------------
torch::Tensor two_crop_augment(torch::Tensor src, torch::Tensor params,
                               int64_t S, bool out_bf16, bool channels_last) {
  CHECK_CUDA_CONTIG(src);
  CHECK_CUDA_CONTIG(params);
  TORCH_CHECK((src.scalar_type() == torch::kFloat32 ||
               src.scalar_type() == torch::kUInt8) &&
              src.dim() == 4 && src.size(1) == 3,
              "src must be fp32 or uint8 [B,3,H,W]");
  TORCH_CHECK(params.scalar_type() == torch::kFloat32 &&
              params.size(1) == 12);
  const int64_t B = src.size(0), H = src.size(2), W = src.size(3);
  const int64_t M = params.size(0);
  at::cuda::CUDAGuard guard(src.device());
  // workspaces/out are fp32/bf16 regardless of the (possibly uint8) source
  auto f32 = src.options().dtype(torch::kFloat32);
  auto out_opts = out_bf16 ? f32.dtype(torch::kBFloat16) : f32;
  torch::Tensor out = torch::empty({M, 3, S, S}, out_opts);
  if (channels_last)
    out = out.contiguous(torch::MemoryFormat::ChannelsLast);
  auto tmp1 = torch::empty({M, 3, S, S}, f32);
  auto tmp2 = torch::empty({M, 3, S, S}, f32);
  auto graypart = torch::empty({M, (S * S + 255) / 256}, f32);
  CHECK_LAUNCH(launch_two_crop_augment(
      cur_stream(), src.data_ptr(),
      src.scalar_type() == torch::kUInt8, params.data_ptr<float>(),
      out.data_ptr(), tmp1.data_ptr<float>(), tmp2.data_ptr<float>(),
      graypart.data_ptr<float>(), B, M, H, W, S, out_bf16, channels_last));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  mod.def("l2norm_rows_fwd", &l2norm_rows_fwd);
  mod.def("l2norm_rows_bwd", &l2norm_rows_bwd);
  mod.def("contrastive_fwd", &contrastive_fwd);
  mod.def("contrastive_bwd", &contrastive_bwd);
  mod.def("softmax_ce0_fwd", &softmax_ce0_fwd);
  mod.def("softmax_ce0_bwd", &softmax_ce0_bwd, py::arg("logits"),
          py::arg("row_max"), py::arg("row_lse"), py::arg("scale"),
          py::arg("gscale") = c10::nullopt);
  mod.def("queue_enqueue", &queue_enqueue);
  mod.def("queue_enqueue_dev", &queue_enqueue_dev);
  mod.def("multi_tensor_ema", &multi_tensor_ema);
  mod.def("multi_cast_bf16", &multi_cast_bf16);
  mod.def("multi_transpose_bf16", &multi_transpose_bf16);
  mod.def("multi_tensor_sgd", &multi_tensor_sgd);
  mod.def("ema_flat", &ema_flat);
  mod.def("grad_norm", &grad_norm);
  mod.def("norm_residual", &norm_residual);
  mod.def("adamw_step", &adamw_step);
  mod.def("adamw8bit_values", &adamw8bit_values);
  mod.def("two_crop_augment", &two_crop_augment);
  mod.def("bn_fwd_train", &bn_fwd_train);
  mod.def("bn_fwd_eval", &bn_fwd_eval);
  mod.def("bn_bwd", &bn_bwd);
  mod.def("bn_stats", &bn_stats);
  mod.def("bn_finalize", &bn_finalize, py::arg("ssum"), py::arg("ssq"),
          py::arg("R"), py::arg("rmean"), py::arg("rvar"), py::arg("eps"),
          py::arg("momentum"), py::arg("zero_src") = false);
  mod.def("bn_bwd_dx_only", &bn_bwd_dx_only);
  mod.def("maxpool_fwd", &maxpool_fwd);
  mod.def("gemm_nt_bf16", &gemm_nt_bf16, py::arg("A"), py::arg("Bt"),
          py::arg("c_add") = c10::nullopt);
  mod.def("gemm_nt_fp8", &gemm_nt_fp8, py::arg("A"), py::arg("Bt"),
          py::arg("out_scale"), py::arg("want_stats") = false,
          py::arg("ws_sum") = c10::nullopt, py::arg("ws_ssq") = c10::nullopt);
  mod.def("gemm_nt_fused", &gemm_nt_fused, py::arg("A"), py::arg("Bt"),
          py::arg("a_scale"), py::arg("a_shift"), py::arg("a_relu"),
          py::arg("want_stats"), py::arg("want_aout") = false,
          py::arg("c_add") = c10::nullopt,
          py::arg("ws_sum") = c10::nullopt,
          py::arg("ws_ssq") = c10::nullopt);
  mod.def("conv3x3_fwd", &conv3x3_fwd);
  mod.def("conv1x1_strided", &conv1x1_strided);
  mod.def("gemm_nt_dgrad_epi", &gemm_nt_dgrad_epi, py::arg("A"),
          py::arg("Bt"), py::arg("y"), py::arg("z"), py::arg("mean"),
          py::arg("rstd"), py::arg("c_add") = c10::nullopt,
          py::arg("ws_db") = c10::nullopt, py::arg("ws_dg") = c10::nullopt);
  mod.def("maxpool_bwd", &maxpool_bwd);
  mod.def("avgpool_fwd", &avgpool_fwd);
  mod.def("avgpool_bwd", &avgpool_bwd);
}
