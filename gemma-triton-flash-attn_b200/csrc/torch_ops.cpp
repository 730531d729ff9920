// torch operators over the C ABI (include/gqa_fa_b200.h): torch.ops.gqafa.fwd,
// torch.ops.gqafa.bwd, and the paged 4-bit cache's kv4_plan, kv4_append,
// kv4_read and kv4_attend.
//
// These are the launch sites of the reference's autograd function
// (flash_attn/attention.py:1435-1473 forward, :1476-1622 backward) as
// dispatcher operators: they allocate the outputs the reference allocates
// (O, LSE; dQ, dK, dV and the delta scratch), pass the current CUDA stream of
// the input's device and turn a non-zero status into the Python exception the
// reference's callers expect (ValueError / NotImplementedError /
// RuntimeError). Compared with calling the C ABI through ctypes this removes
// the per-call Python marshalling of ~30 arguments and stride arrays. No CUDA
// code is compiled here: every kernel lives in libgqa_fa_b200.so.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <string>
#include <tuple>

#include "../../include/gqa_fa_b200.h"

namespace {

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kHalf) return GQAFA_DTYPE_FP16;
  if (t.scalar_type() == at::kBFloat16) return GQAFA_DTYPE_BF16;
  TORCH_CHECK_NOT_IMPLEMENTED(false, "gqafa: dtype ", t.scalar_type(), " is not supported (fp16, bf16)");
  return -1;
}

void check(int rc) {
  if (rc == GQAFA_OK) return;
  const char* msg = gqafa_last_error();
  TORCH_CHECK_NOT_IMPLEMENTED(rc != GQAFA_ERR_UNSUPPORTED, msg);
  TORCH_CHECK_VALUE(rc != GQAFA_ERR_INVALID, msg);
  TORCH_CHECK(false, "gqafa: ", msg);
}

void check_4d(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 4, "gqafa: ", name, " must be 4-D (B, H, N, D)");
  TORCH_CHECK(t.is_cuda(), "gqafa: ", name, " must be a CUDA tensor (there is no CPU path)");
}

// A layout the tensor maps accept: last stride 1, other strides multiples of 8
// elements (size-1 dimensions excepted), 16-byte aligned data. Otherwise a
// contiguous copy, as the Python layer does.
at::Tensor abi_ready(const at::Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3 && ok; ++i) ok = (t.stride(i) % 8 == 0) || t.size(i) == 1;
  return ok ? t : t.contiguous();
}

struct Strides {
  long long s[4];
  explicit Strides(const at::Tensor& t) {
    for (int i = 0; i < 4; ++i) s[i] = t.stride(i);
  }
};

std::tuple<at::Tensor, at::Tensor> fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                       bool causal, int64_t window, double scale, bool want_lse) {
  check_4d(q_in, "q");
  check_4d(k_in, "k");
  check_4d(v_in, "v");
  c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = abi_ready(q_in), k = abi_ready(k_in), v = abi_ready(v_in);
  const int64_t B = q.size(0), Hq = q.size(1), N = q.size(2), D = q.size(3), Hkv = k.size(1), Nk = k.size(2);
  at::Tensor o = abi_ready(at::empty_like(q));  // keeps q's layout (HF's (B, N, H, D) storage)
  at::Tensor lse = want_lse ? at::empty({B, Hq, N}, q.options().dtype(at::kFloat)) : at::Tensor();
  const Strides sq(q), sk(k), sv(v), so(o);
  void* stream = c10::cuda::getCurrentCUDAStream(q.get_device()).stream();
  float* lp = want_lse ? lse.data_ptr<float>() : nullptr;
  int rc;
  if (Nk == N) {
    rc = gqafa_fwd(q.data_ptr(), sq.s, k.data_ptr(), sk.s, v.data_ptr(), sv.s, o.data_ptr(), so.s, lp, (int)B,
                   (int)Hq, (int)Hkv, (int)N, (int)D, (float)scale, causal ? 1 : 0, (int)window, dtype_code(q),
                   stream);
  } else {
    rc = gqafa_fwd_kv(q.data_ptr(), sq.s, k.data_ptr(), sk.s, v.data_ptr(), sv.s, o.data_ptr(), so.s, lp, (int)B,
                      (int)Hq, (int)Hkv, (int)N, (int)Nk, (int)D, (float)scale, causal ? 1 : 0, (int)window,
                      dtype_code(q), stream);
  }
  check(rc);
  return {o, want_lse ? lse : at::empty({0}, q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bwd(const at::Tensor& q_in, const at::Tensor& k_in,
                                                   const at::Tensor& v_in, const at::Tensor& o_in,
                                                   const at::Tensor& lse_in, const at::Tensor& do_in, bool causal,
                                                   int64_t window, double scale,
                                                   const c10::optional<at::Tensor>& workspace) {
  for (auto* t : {&q_in, &k_in, &v_in, &o_in, &do_in}) check_4d(*t, "tensor");
  c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = abi_ready(q_in), k = abi_ready(k_in), v = abi_ready(v_in), o = abi_ready(o_in),
                   dout = abi_ready(do_in), lse = lse_in.contiguous();
  const int64_t B = q.size(0), Hq = q.size(1), N = q.size(2), D = q.size(3), Hkv = k.size(1);
  TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.numel() == B * Hq * N,
                    "gqafa: lse must be float32 (B, H_Q, N)");
  at::Tensor dq = abi_ready(at::empty_like(q)), dk = abi_ready(at::empty_like(k)),
             dv = abi_ready(at::empty_like(v));
  at::Tensor delta = at::empty({B, Hq, N}, q.options().dtype(at::kFloat));
  const Strides sq(q), sk(k), sv(v), so(o), sd(dout), sdq(dq), sdk(dk), sdv(dv);
  void* stream = c10::cuda::getCurrentCUDAStream(q.get_device()).stream();
  int rc;
  if (workspace.has_value() && workspace->defined() && workspace->numel() > 0) {
    const at::Tensor& ws = *workspace;
    TORCH_CHECK_VALUE(ws.is_cuda() && ws.is_contiguous(), "gqafa: workspace must be a contiguous CUDA tensor");
    rc = gqafa_bwd_ws(q.data_ptr(), sq.s, k.data_ptr(), sk.s, v.data_ptr(), sv.s, o.data_ptr(), so.s,
                      dout.data_ptr(), sd.s, lse.data_ptr<float>(), dq.data_ptr(), sdq.s, dk.data_ptr(), sdk.s,
                      dv.data_ptr(), sdv.s, delta.data_ptr<float>(), (int)B, (int)Hq, (int)Hkv, (int)N, (int)D,
                      (float)scale, causal ? 1 : 0, (int)window, dtype_code(q), stream, ws.data_ptr(),
                      (long long)(ws.numel() * ws.element_size()));
  } else {
    rc = gqafa_bwd(q.data_ptr(), sq.s, k.data_ptr(), sk.s, v.data_ptr(), sv.s, o.data_ptr(), so.s, dout.data_ptr(),
                   sd.s, lse.data_ptr<float>(), dq.data_ptr(), sdq.s, dk.data_ptr(), sdk.s, dv.data_ptr(), sdv.s,
                   delta.data_ptr<float>(), (int)B, (int)Hq, (int)Hkv, (int)N, (int)D, (float)scale,
                   causal ? 1 : 0, (int)window, dtype_code(q), stream);
  }
  check(rc);
  return {dq, dk, dv};
}

// Shapes only (no launch), for tracing and fake-tensor propagation.
std::tuple<at::Tensor, at::Tensor> fwd_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool,
                                            int64_t, double, bool want_lse) {
  return {at::empty_like(q),
          at::empty(want_lse ? std::vector<int64_t>{q.size(0), q.size(1), q.size(2)} : std::vector<int64_t>{0},
                    q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bwd_meta(const at::Tensor& q, const at::Tensor& k,
                                                        const at::Tensor& v, const at::Tensor&, const at::Tensor&,
                                                        const at::Tensor&, bool, int64_t, double,
                                                        const c10::optional<at::Tensor>&) {
  return {at::empty_like(q), at::empty_like(k), at::empty_like(v)};
}

// ---------------------------------------------------------------- 4-bit cache
// Device and type checks live here, beside the launch: everything below is
// handed to the C ABI as raw pointers. Messages take numbers as strings: with a
// libstdc++ linked in statically (some toolchains do), writing a number to the
// stream behind TORCH_CHECK mixes two copies of the library and crashes.
std::string str(int64_t v) { return std::to_string(v); }
void check_int32(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda(), "gqafa: ", name, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK_VALUE(t.device() == dev, "gqafa: ", name, " is on ", t.device().str(), ", expected ", dev.str());
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, "gqafa: ", name, " must be int32, got ", c10::toString(t.scalar_type()));
}
at::Tensor vector_int32(const at::Tensor& t, const char* name, int64_t n, const at::Device& dev) {
  check_int32(t, name, dev);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, "gqafa: ", name, " must have shape (", str(n), ",)");
  return t.contiguous();
}
// A matrix whose rows are contiguous (any row stride).
at::Tensor rows_int32(const at::Tensor& t, const char* name, int64_t rows, const at::Device& dev) {
  check_int32(t, name, dev);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) > 0, "gqafa: ", name, " must have shape (",
                    str(rows), ", n > 0)");
  return (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= 0 ? t : t.contiguous();
}
struct Pages {
  int64_t count, heads, page_size, dim;
};
Pages check_pages(const at::Tensor& pages, int64_t page_size, const at::Device& dev) {
  TORCH_CHECK(pages.is_cuda(), "gqafa: pages must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK_VALUE(pages.device() == dev, "gqafa: pages are on ", pages.device().str(), ", expected ", dev.str());
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kByte && pages.dim() == 5 && pages.is_contiguous() && pages.size(1) == 2,
                    "gqafa: pages must be a contiguous uint8 tensor (pages, 2, heads, blocks, block bytes)");
  TORCH_CHECK_VALUE(page_size == 16 * pages.size(3), "gqafa: pages hold ", str(16 * pages.size(3)),
                    " tokens each, page_size is ", str(page_size));
  const int64_t dim = pages.size(4) / 544 * 64;
  TORCH_CHECK_VALUE(pages.size(4) % 544 == 0 && dim > 0, "gqafa: a block of pages must hold 544 bytes per 64 dims");
  return {pages.size(0), pages.size(2), page_size, dim};
}
void check_rows(const at::Tensor& t, const char* name, const Pages& pg, const at::Device& dev) {
  check_4d(t, name);
  TORCH_CHECK_VALUE(t.device() == dev, "gqafa: ", name, " is on ", t.device().str(), ", expected ", dev.str());
  TORCH_CHECK_VALUE(t.size(3) == pg.dim, "gqafa: ", name, " has head_dim ", str(t.size(3)), ", the cache ",
                    str(pg.dim));
  TORCH_CHECK_VALUE(t.numel() > 0, "gqafa: ", name, " is empty");
}
// As abi_ready, and a broadcast tensor (stride 0) becomes a whole one.
at::Tensor rows_ready(const at::Tensor& t) {
  bool ok = true;
  for (int i = 0; i < 3; ++i) ok = ok && (t.stride(i) > 0 || t.size(i) == 1);
  return abi_ready(ok ? t : t.contiguous());
}
// Outputs and scratch of these operators come from the caching allocator
// directly: a step of a few microseconds on the GPU would otherwise wait for
// the dispatcher's at::empty, 1.6 us a tensor (the plan has seven).
at::Tensor new_tensor(at::IntArrayRef size, at::ScalarType type) {
  return at::detail::empty_generic(size, c10::cuda::CUDACachingAllocator::get(),
                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}
at::Tensor new_like(const at::Tensor& t) {  // with t's layout where it is dense (HF's (B, N, H, D) storage)
  if (!t.is_non_overlapping_and_dense()) return new_tensor(t.sizes(), t.scalar_type());
  return at::detail::empty_strided_generic(t.sizes(), t.strides(), c10::cuda::CUDACachingAllocator::get(),
                                           c10::DispatchKeySet(c10::DispatchKey::CUDA), t.scalar_type());
}
// Contiguous int32 tensors cut from one allocation, each 16-byte aligned.
class Int32Pack {
 public:
  explicit Int32Pack(int64_t ints) {
    auto* alloc = c10::cuda::CUDACachingAllocator::get();
    const size_t bytes = static_cast<size_t>(ints) * 4;
    storage_ = c10::Storage(c10::Storage::use_byte_size_t(), bytes, alloc->allocate(bytes), alloc, false);
  }
  static int64_t room(int64_t n) { return (n + 3) / 4 * 4; }
  at::Tensor cut(at::IntArrayRef size) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(storage_), c10::DispatchKeySet(c10::DispatchKey::CUDA), caffe2::TypeMeta::Make<int32_t>());
    t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
    t.unsafeGetTensorImpl()->set_storage_offset(at_);
    at_ += room(t.numel());
    return t;
  }

 private:
  c10::Storage storage_;
  int64_t at_ = 0;
};
int to_int(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, "gqafa: ", name, " out of range: ", str(v));
  return static_cast<int>(v);
}

using Plan = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Plan kv4_plan(const at::Tensor& kv_lens, const at::Tensor& new_lens, const at::Tensor& block_table,
              at::Tensor free_pages, const at::Tensor& free_state, int64_t page_size, int64_t max_new) {
  const at::Device dev = kv_lens.device();
  TORCH_CHECK(kv_lens.is_cuda(), "gqafa: kv_lens must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK_VALUE(kv_lens.dim() == 1 && kv_lens.size(0) > 0, "gqafa: kv_lens must have shape (B > 0,)");
  TORCH_CHECK_VALUE(max_new > 0, "gqafa: max_new must be positive");
  c10::cuda::CUDAGuard guard(dev);
  const int64_t B = kv_lens.size(0);
  const at::Tensor lens = vector_int32(kv_lens, "kv_lens", B, dev), add = vector_int32(new_lens, "new_lens", B, dev),
                   state = vector_int32(free_state, "free_state", 2, dev),
                   table = rows_int32(block_table, "block_table", B, dev);
  check_int32(free_pages, "free_pages", dev);
  TORCH_CHECK_VALUE(free_pages.dim() == 1 && free_pages.size(0) > 0 && free_pages.is_contiguous(),
                    "gqafa: free_pages must be a contiguous vector (it is written to)");
  const int64_t cols = table.size(1);
  Int32Pack pack(Int32Pack::room(B * cols) + 2 * Int32Pack::room(B * max_new) + 3 * Int32Pack::room(B) + 4);
  at::Tensor out_table = pack.cut({B, cols}), slots = pack.cut({B, max_new}), positions = pack.cut({B, max_new}),
             out_lens = pack.cut({B}), out_new = pack.cut({B}), accepted = pack.cut({B}), out_state = pack.cut({2});
  check(gqafa_kv4_plan(lens.data_ptr<int>(), add.data_ptr<int>(), table.data_ptr<int>(), table.stride(0),
                       free_pages.data_ptr<int>(), state.data_ptr<int>(), to_int(B, "B"), to_int(cols, "columns"),
                       to_int(free_pages.size(0), "free_pages"), to_int(page_size, "page_size"),
                       to_int(max_new, "max_new"), out_table.data_ptr<int>(), out_lens.data_ptr<int>(),
                       out_new.data_ptr<int>(), slots.data_ptr<int>(), positions.data_ptr<int>(),
                       accepted.data_ptr<int>(), out_state.data_ptr<int>(),
                       c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {out_table, out_lens, out_new, slots, positions, out_state, accepted};
}

void kv4_append(at::Tensor pages, const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& slot_map,
                int64_t page_size) {
  const at::Device dev = k_in.device();
  const Pages pg = check_pages(pages, page_size, dev);
  check_rows(k_in, "k", pg, dev);
  check_rows(v_in, "v", pg, dev);
  TORCH_CHECK_VALUE(k_in.sizes() == v_in.sizes() && k_in.size(1) == pg.heads,
                    "gqafa: k and v must have shape (B, ", str(pg.heads), ", N, ", str(pg.dim), ")");
  TORCH_CHECK_TYPE(k_in.scalar_type() == v_in.scalar_type(), "gqafa: k and v must share a dtype");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor k = rows_ready(k_in), v = rows_ready(v_in);
  const int64_t B = k.size(0), N = k.size(2);
  const at::Tensor slots = rows_int32(slot_map, "slot_map", B, dev);
  TORCH_CHECK_VALUE(slots.size(1) == N, "gqafa: slot_map must have shape (", str(B), ", ", str(N), ")");
  const Strides sk(k), sv(v);
  check(gqafa_kv4_append(k.data_ptr(), sk.s, v.data_ptr(), sv.s, slots.data_ptr<int>(), slots.stride(0),
                         pages.data_ptr(), pg.count, to_int(B, "B"), to_int(pg.heads, "heads"), to_int(N, "N"),
                         to_int(pg.dim, "head_dim"), to_int(page_size, "page_size"), dtype_code(k),
                         c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
}

std::tuple<at::Tensor, at::Tensor> kv4_read(const at::Tensor& pages, const at::Tensor& block_table,
                                            const at::Tensor& kv_lens, int64_t n,
                                            const c10::optional<at::Tensor>& starts, int64_t page_size,
                                            at::ScalarType dtype) {
  const at::Device dev = pages.device();
  const Pages pg = check_pages(pages, page_size, dev);
  TORCH_CHECK_VALUE(n > 0, "gqafa: the number of rows must be positive");
  TORCH_CHECK_VALUE(kv_lens.dim() == 1 && kv_lens.size(0) > 0, "gqafa: kv_lens must have shape (B > 0,)");
  c10::cuda::CUDAGuard guard(dev);
  const int64_t B = kv_lens.size(0);
  const at::Tensor lens = vector_int32(kv_lens, "kv_lens", B, dev), table = rows_int32(block_table, "block_table", B, dev);
  at::Tensor from;
  if (starts.has_value() && starts->defined()) from = vector_int32(*starts, "starts", B, dev);
  at::Tensor k = new_tensor({B, pg.heads, n, pg.dim}, dtype), v = new_tensor({B, pg.heads, n, pg.dim}, dtype);
  check(gqafa_kv4_read(pages.data_ptr(), pg.count, table.data_ptr<int>(), table.stride(0),
                       to_int(table.size(1), "columns"), lens.data_ptr<int>(),
                       from.defined() ? from.data_ptr<int>() : nullptr, k.data_ptr(), v.data_ptr(), to_int(B, "B"),
                       to_int(pg.heads, "heads"), to_int(n, "rows"), to_int(pg.dim, "head_dim"),
                       to_int(page_size, "page_size"), dtype_code(k),
                       c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {k, v};
}

std::tuple<at::Tensor, at::Tensor> kv4_attend(const at::Tensor& q_in, const at::Tensor& pages,
                                              const at::Tensor& block_table, const at::Tensor& kv_lens,
                                              const c10::optional<at::Tensor>& q_lens, int64_t page_size,
                                              int64_t max_kv_len, bool causal, int64_t window, double scale,
                                              bool want_lse) {
  const at::Device dev = q_in.device();
  const Pages pg = check_pages(pages, page_size, dev);
  check_rows(q_in, "q", pg, dev);
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = rows_ready(q_in);
  const int64_t B = q.size(0), Hq = q.size(1), N = q.size(2);
  const at::Tensor lens = vector_int32(kv_lens, "kv_lens", B, dev), table = rows_int32(block_table, "block_table", B, dev);
  at::Tensor rows;
  if (q_lens.has_value() && q_lens->defined()) rows = vector_int32(*q_lens, "q_lens", B, dev);
  at::Tensor o = new_like(q);
  at::Tensor lse = new_tensor({want_lse ? B : 0, Hq, N}, at::kFloat);
  const int b = to_int(B, "B"), hq = to_int(Hq, "H_Q"), hkv = to_int(pg.heads, "H_KV"), n = to_int(N, "N"),
            d = to_int(pg.dim, "head_dim"), win = to_int(causal ? window : 0, "window");
  const int64_t capacity = table.size(1) * page_size;
  const int longest = to_int(max_kv_len > 0 && max_kv_len < capacity ? max_kv_len : capacity, "max_kv_len");
  const long long bytes = gqafa_kv4_attend_workspace_size(b, hq, hkv, n, d, longest, win);
  if (bytes < 0) {
    const char* msg = gqafa_last_error();
    TORCH_CHECK_NOT_IMPLEMENTED(d == 64 || d == 128 || d == 256 || d == 512, msg);
    TORCH_CHECK_VALUE(false, msg);
  }
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  const Strides sq(q), so(o);
  check(gqafa_kv4_attend(q.data_ptr(), sq.s, pages.data_ptr(), pg.count, table.data_ptr<int>(), table.stride(0),
                         to_int(table.size(1), "columns"), lens.data_ptr<int>(),
                         rows.defined() ? rows.data_ptr<int>() : nullptr, o.data_ptr(), so.s,
                         want_lse ? lse.data_ptr<float>() : nullptr, b, hq, hkv, n, d, to_int(page_size, "page_size"),
                         longest, (float)scale, causal ? 1 : 0, win, dtype_code(q), ws.get(), bytes,
                         c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {o, lse};
}

Plan kv4_plan_meta(const at::Tensor& kv_lens, const at::Tensor&, const at::Tensor& table, at::Tensor, const at::Tensor&,
                   int64_t, int64_t max_new) {
  const auto opt = kv_lens.options();
  const auto B = kv_lens.size(0);
  return {at::empty({B, table.size(1)}, opt), at::empty({B}, opt),       at::empty({B}, opt), at::empty({B, max_new}, opt),
          at::empty({B, max_new}, opt),       at::empty({2}, opt), at::empty({B}, opt)};
}
void kv4_append_meta(at::Tensor, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t) {}
std::tuple<at::Tensor, at::Tensor> kv4_read_meta(const at::Tensor& pages, const at::Tensor&, const at::Tensor& lens,
                                                 int64_t n, const c10::optional<at::Tensor>&, int64_t,
                                                 at::ScalarType dtype) {
  at::Tensor k = at::empty({lens.size(0), pages.size(2), n, pages.size(4) / 544 * 64}, pages.options().dtype(dtype));
  return {k, at::empty_like(k)};
}
std::tuple<at::Tensor, at::Tensor> kv4_attend_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                   const at::Tensor&, const c10::optional<at::Tensor>&, int64_t,
                                                   int64_t, bool, int64_t, double, bool want_lse) {
  return {at::empty_like(q),
          at::empty({want_lse ? q.size(0) : 0, q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

}  // namespace

TORCH_LIBRARY(gqafa, m) {
  m.def("fwd(Tensor q, Tensor k, Tensor v, bool causal, int window, float scale, bool want_lse) -> (Tensor, Tensor)");
  m.def(
      "bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, bool causal, int window, float scale, "
      "Tensor? workspace) -> (Tensor, Tensor, Tensor)");
  m.def(
      "kv4_plan(Tensor kv_lens, Tensor new_lens, Tensor block_table, Tensor(a!) free_pages, Tensor free_state, "
      "int page_size, int max_new) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("kv4_append(Tensor(a!) pages, Tensor k, Tensor v, Tensor slot_map, int page_size) -> ()");
  m.def(
      "kv4_read(Tensor pages, Tensor block_table, Tensor kv_lens, int n, Tensor? starts, int page_size, "
      "ScalarType dtype) -> (Tensor, Tensor)");
  m.def(
      "kv4_attend(Tensor q, Tensor pages, Tensor block_table, Tensor kv_lens, Tensor? q_lens, int page_size, "
      "int max_kv_len, bool causal, int window, float scale, bool want_lse) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gqafa, CUDA, m) {
  m.impl("fwd", &fwd);
  m.impl("bwd", &bwd);
  m.impl("kv4_plan", &kv4_plan);
  m.impl("kv4_append", &kv4_append);
  m.impl("kv4_read", &kv4_read);
  m.impl("kv4_attend", &kv4_attend);
}

TORCH_LIBRARY_IMPL(gqafa, Meta, m) {
  m.impl("fwd", &fwd_meta);
  m.impl("bwd", &bwd_meta);
  m.impl("kv4_plan", &kv4_plan_meta);
  m.impl("kv4_append", &kv4_append_meta);
  m.impl("kv4_read", &kv4_read_meta);
  m.impl("kv4_attend", &kv4_attend_meta);
}
