// Host side of the block operators: argument checks, strided views, output and
// workspace buffers, and the call of the C ABI on the current stream.
//
// A Python extension over torch's tensors.  In Python the same steps took 10 to
// 16 us of a call, which for a single token is four times the kernel.  The
// entry points of libvcattn.so come in as addresses (bind), from the handle
// that the ctypes binding has loaded.
#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/extension.h>

#include <atomic>
#include <memory>
#include <mutex>
#include <optional>
#include <sstream>
#include <string>
#include <vector>

#include "vcattn.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// What one loaded copy of the package brings: the library's entry points and
// its `check`, which raises that copy's VCAttnError with the library's message.
struct Library {
  decltype(&vcattn_qk_norm_rope) qk_norm_rope = nullptr;
  decltype(&vcattn_quantize_blocks) quantize_blocks = nullptr;
  decltype(&vcattn_matmul_blocks) matmul_blocks = nullptr;
  decltype(&vcattn_matmul_blocks_workspace_bytes) matmul_workspace = nullptr;
  decltype(&vcattn_attn_packed) attn_packed = nullptr;
  py::object check;

  void status(int rc, const char* fn) const {
    if (rc != VCATTN_OK) check(fn, rc);
  }
};

template <typename F> void address(const py::dict& d, const char* name, F& f) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}

// ---- errors -------------------------------------------------------------------
template <typename... A> std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
#define CHECK_VALUE(cond, ...) \
  do {                         \
    if (!(cond)) throw py::value_error(text(__VA_ARGS__)); \
  } while (0)

void need_cuda(bool cuda, const char* fn) {
  if (!cuda) throw std::runtime_error(text(fn, " needs CUDA tensors (this build has no CPU path)"));
}

// The operators have no derivatives, backward or forward (a tangent sits on the
// tensor whatever the gradient mode): say so instead of dropping them.
void refuse_one(const char* fn, const Tensor& t) {
  if (!t.defined()) return;
  if (t.requires_grad() && at::GradMode::is_enabled())
    throw std::runtime_error(text(fn, " has no backward pass: call it under torch.no_grad() or on detached tensors"));
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined())
    throw std::runtime_error(text(fn, " has no forward derivative: call it on detached tensors"));
}
void refuse_one(const char* fn, const OptTensor& t) {
  if (t.has_value()) refuse_one(fn, *t);
}
template <typename... T> void refuse_grad(const char* fn, const T&... t) { (refuse_one(fn, t), ...); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return VCATTN_DTYPE_BF16;
    case at::kHalf: return VCATTN_DTYPE_F16;
    case at::kFloat: return VCATTN_DTYPE_F32;
    default: throw py::type_error(text("unsupported dtype ", t));
  }
}

bool aligned(const void* p, int64_t bytes = 0) { return ((reinterpret_cast<uintptr_t>(p) | bytes) & 15) == 0; }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ---- views ----------------------------------------------------------------------
// vcattn_bhnd of a (B, H, N, D) tensor and the tensor it points into: a copy if
// the channels are not contiguous, a row is not on a 16-byte boundary or rows
// are the same memory (a broadcast view).
struct View {
  vcattn_bhnd v;
  Tensor keep;
};
vcattn_bhnd bhnd(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
View view(const Tensor& t) {
  const int64_t rows = t.stride(0) | t.stride(1) | t.stride(2);
  if (t.stride(3) == 1 && aligned(t.data_ptr(), rows * t.element_size()) && t.stride(0) && t.stride(1) && t.stride(2))
    return {bhnd(t), t};
  Tensor c = t.clone(at::MemoryFormat::Contiguous);
  return {bhnd(c), c};
}

// Outputs that the caller gives may not share memory with a tensor that the
// kernel reads at other places, or at other times, than it writes.  (Two views
// that interleave, as those of a fused projection, are told apart only where
// they start at the same element.)
bool same_start(const Tensor& x, const Tensor& y) { return x.numel() > 0 && y.numel() > 0 && x.data_ptr() == y.data_ptr(); }
void apart(const Tensor& out, const Tensor& in, const char* what, const char* other) {
  const at::MemOverlapStatus o = at::get_overlap_status(out, in);
  CHECK_VALUE(o != at::MemOverlapStatus::Full && o != at::MemOverlapStatus::Partial && !same_start(out, in), what,
              " overlaps ", other);
}
// The same for the input that it may be written over.
void in_place_or_apart(const Tensor& out, const Tensor& in, const char* what, const char* other) {
  CHECK_VALUE(at::get_overlap_status(out, in) != at::MemOverlapStatus::Partial &&
                  (!same_start(out, in) || out.strides() == in.strides()),
              what, " overlaps a part of ", other);
}

// Tells autograd that `t` has new contents, so that a backward pass which needs
// the old ones refuses instead of using these.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// `out` checked against its input, or a new buffer with its dimensions in the
// input's order in memory (the ComfyUI (B, N, H*D) path stays token-major).
Tensor out_rows(const OptTensor& out, const Tensor& x, const char* what) {
  if (!out.has_value()) {
    Tensor t = at::empty_like(x);
    return t.stride(3) == 1 ? t : at::empty(x.sizes(), x.options());
  }
  const Tensor& t = *out;
  CHECK_VALUE(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device(), what,
              " must match its input: ", x.sizes(), " ", x.scalar_type(), " on ", x.device());
  if (t.numel() > 0) {
    const int64_t rows = t.stride(0) | t.stride(1) | t.stride(2);
    bool own = t.stride(3) == 1 && aligned(t.data_ptr(), rows * t.element_size());
    for (int i = 0; i < 4; ++i) own &= t.stride(i) != 0 || t.size(i) == 1;
    CHECK_VALUE(own, what, " must have contiguous channels and 16-byte aligned rows of their own");
  }
  return t;
}

// ---- qk_norm_rope -----------------------------------------------------------------
// A (D,) weight as the kernel reads it: fp32, contiguous, 16-byte aligned.
const float* weight(const OptTensor& w, int64_t d, const at::Device& dev, const char* what, Tensor& keep) {
  if (!w.has_value()) return nullptr;
  CHECK_VALUE(w->dim() == 1 && w->size(0) == d, what, " must be (", d, ",), got ", w->sizes());
  CHECK_VALUE(w->device() == dev, what, " must be on ", dev, ", got ", w->device());
  keep = w->scalar_type() == at::kFloat ? *w : w->to(at::kFloat);
  if (keep.stride(0) != 1 || !aligned(keep.data_ptr())) keep = keep.clone(at::MemoryFormat::Contiguous);
  return static_cast<const float*>(keep.data_ptr());
}

constexpr int64_t kMaxRows = (int64_t{1} << 31) - 1;

std::tuple<Tensor, Tensor> qk_norm_rope(const Library& lib, const Tensor& q, const Tensor& k, const OptTensor& cos_in, const OptTensor& sin_in,
                                        const OptTensor& q_weight, const OptTensor& k_weight, const std::string& layout,
                                        double eps, bool norm, const OptTensor& out_q, const OptTensor& out_k) {
  refuse_grad("qk_norm_rope", q, k, cos_in, sin_in, q_weight, k_weight, out_q, out_k);
  need_cuda(q.is_cuda() && k.is_cuda(), "qk_norm_rope");
  CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
              "q and k must be (B, Hq, N, D) and (B, Hk, N, D), got ", q.sizes(), ", ", k.sizes());
  const at::Device dev = q.device();
  CHECK_VALUE(q.scalar_type() == k.scalar_type() && k.device() == dev, "q and k must share a dtype and a device");
  const int dt = dtype_code(q.scalar_type());
  const int64_t b = q.size(0), n = q.size(2), d = q.size(3);
  CHECK_VALUE(d % 8 == 0 && d >= 8 && d <= 256, "head_dim must be a multiple of 8 up to 256, got ", d);
  // (the C entry point takes these as int: checked here, before they are narrowed)
  const int64_t heads = q.size(1) + k.size(1);
  CHECK_VALUE(b <= kMaxRows && n <= kMaxRows && heads <= kMaxRows && b * n <= kMaxRows / std::max<int64_t>(heads, 1),
              "2^31 head rows or more: q ", q.sizes(), ", k ", k.sizes());
  CHECK_VALUE(layout == "half" || layout == "interleaved", "layout must be 'half' or 'interleaved', got '", layout, "'");
  const int flags = (layout == "half" ? 0 : VCATTN_ROPE_INTERLEAVED) | (norm ? VCATTN_ROPE_NORM : 0);
  CHECK_VALUE(cos_in.has_value() == sin_in.has_value(), "cos and sin are given together");
  Tensor cos, sin, wq, wk;
  int64_t rot = 0, tsb = 0, tsn = 0;
  if (cos_in.has_value()) {
    cos = *cos_in;
    sin = *sin_in;
    const int64_t t = cos.dim();
    CHECK_VALUE(cos.sizes() == sin.sizes() && (t == 2 || t == 3) && cos.size(t - 2) == n &&
                    (t == 2 || cos.size(0) == 1 || cos.size(0) == b),
                "cos and sin must be (", n, ", r/2) or (", b, ", ", n, ", r/2), got ", cos.sizes(), ", ", sin.sizes());
    CHECK_VALUE(cos.device() == dev && sin.device() == dev, "cos and sin must be on ", dev);
    rot = 2 * cos.size(t - 1);
    CHECK_VALUE(rot % 16 == 0 && rot <= d, "the rotated channels must be a multiple of 16 up to ", d, ", got ", rot);
    if (cos.scalar_type() != at::kFloat) cos = cos.to(at::kFloat);
    if (sin.scalar_type() != at::kFloat) sin = sin.to(at::kFloat);
    const int64_t rows = cos.stride(t - 2) | (t == 3 ? cos.stride(0) : 0);
    if (cos.strides() != sin.strides() || cos.stride(t - 1) != 1 || !aligned(cos.data_ptr(), rows * 4) ||
        !aligned(sin.data_ptr())) {
      cos = cos.clone(at::MemoryFormat::Contiguous);
      sin = sin.clone(at::MemoryFormat::Contiguous);
    }
    tsn = cos.stride(t - 2);
    tsb = t == 3 && cos.size(0) > 1 ? cos.stride(0) : 0;
  }
  const float* qw = weight(q_weight, d, dev, "q_weight", wq);
  const float* kw = weight(k_weight, d, dev, "k_weight", wk);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor oq = out_rows(out_q, q, "out[0]"), ok = out_rows(out_k, k, "out[1]");
  if (out_q.has_value()) {
    in_place_or_apart(oq, q, "out[0]", "q");
    apart(oq, k, "out[0]", "k");
  }
  if (out_k.has_value()) {
    in_place_or_apart(ok, k, "out[1]", "k");
    apart(ok, q, "out[1]", "q");
    apart(ok, oq, "out[1]", "out[0]");
  }
  const View vq = view(q), vk = view(k);
  const vcattn_bhnd wq_out = bhnd(oq), wk_out = bhnd(ok);
  lib.status(lib.qk_norm_rope(&vq.v, &vk.v, dt, static_cast<int>(b), static_cast<int>(q.size(1)),
                                  static_cast<int>(k.size(1)), static_cast<int>(n), static_cast<int>(d), qw, kw,
                                  rot ? static_cast<const float*>(cos.data_ptr()) : nullptr,
                                  rot ? static_cast<const float*>(sin.data_ptr()) : nullptr, tsb, tsn,
                                  static_cast<int>(rot), flags, static_cast<float>(eps), &wq_out, &wk_out, stream_of(q)),
               "vcattn_qk_norm_rope");
  if (out_q.has_value()) written(oq);
  if (out_k.has_value()) written(ok);
  return {oq, ok};
}

// ---- quantize_blocks --------------------------------------------------------------
constexpr int64_t kBlock = 128;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

std::tuple<Tensor, Tensor> quantize_blocks(const Library& lib, const Tensor& x, int64_t rows) {
  refuse_grad("quantize_blocks", x);
  need_cuda(x.is_cuda(), "quantize_blocks");
  CHECK_VALUE(rows == 1 || rows == kBlock, "rows must be 1 or ", kBlock, ", got ", rows);
  const int dt = dtype_code(x.scalar_type());
  CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must be (M, K) with K > 0, got ", x.sizes());
  const int64_t k = x.size(-1);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
  const int64_t m = x2.size(0);
  if ((x2.stride(1) != 1 && k > 1) || (m > 1 && x2.stride(0) < k)) x2 = x2.clone(at::MemoryFormat::Contiguous);
  const int64_t ldx = std::max(x2.stride(0), k), ldc = ceil_div(k, 16) * 16, mb = ceil_div(m, rows);
  // (code rows 16 bytes apart at least, scales with rows side by side)
  const Tensor codes = at::empty_strided({m, k}, {ldc, 1}, x.options().dtype(at::kFloat8_e4m3fn));
  const Tensor scale = at::empty_strided({mb, ceil_div(k, kBlock)}, {1, mb}, x.options().dtype(at::kFloat));
  lib.status(lib.quantize_blocks(x2.data_ptr(), dt, m, k, ldx, static_cast<int>(rows),
                                     static_cast<uint8_t*>(codes.data_ptr()), ldc, static_cast<float*>(scale.data_ptr()),
                                     1, mb, stream_of(x)),
               "vcattn_quantize_blocks");
  return {codes, scale};
}

// ---- matmul_blocks ----------------------------------------------------------------
// Checked codes as the TMA reads them (16-byte rows, copied if need be) and their pitch.
Tensor code_rows(const Tensor& c, const Tensor& s, int64_t rows, int64_t want, const char* name, int64_t& ld) {
  if (!(c.is_cuda() && s.is_cuda()) || c.device() != s.device())
    throw std::runtime_error(text("matmul_blocks needs CUDA tensors on one device (", name, ")"));
  CHECK_VALUE(rows == want, name, " must have one scale per ", want, " row(s) and ", kBlock, " columns, got rows=", rows);
  CHECK_VALUE(c.scalar_type() == at::kFloat8_e4m3fn && c.dim() == 2 && c.size(1) > 0, name,
              ".codes must be (rows, K) float8_e4m3fn, got ", c.sizes(), " ", c.scalar_type());
  const int64_t m = c.size(0), k = c.size(1), sm = ceil_div(m, rows), sk = ceil_div(k, kBlock);
  CHECK_VALUE(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == sm && s.size(1) == sk, name, ".scale must be (",
              sm, ", ", sk, ") float32, got ", s.sizes(), " ", s.scalar_type());
  const int64_t tight = ceil_div(k, 16) * 16;
  ld = m > 1 ? c.stride(0) : tight;   // (the pitch of a single row is never used)
  if ((c.stride(1) == 1 || k == 1) && aligned(c.data_ptr(), ld) && ld >= k) return c;
  ld = tight;
  Tensor t = at::empty_strided({m, k}, {ld, 1}, c.options());
  t.copy_(c);
  return t;
}

Tensor matmul_blocks(const Library& lib, const Tensor& a, const Tensor& sa, int64_t a_rows, const Tensor& b, const Tensor& sb, int64_t b_rows,
                     const OptTensor& bias_in, const py::object& dtype, const OptTensor& out_in) {
  refuse_grad("matmul_blocks", a, sa, b, sb, bias_in, out_in);
  int64_t lda = 0, ldb = 0;
  c10::cuda::OptionalCUDAGuard guard;
  if (a.is_cuda()) guard.set_device(a.device());
  const Tensor ac = code_rows(a, sa, a_rows, 1, "a", lda), bc = code_rows(b, sb, b_rows, kBlock, "b", ldb);
  const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
  const at::Device dev = a.device();
  CHECK_VALUE(b.size(1) == k && b.device() == dev, "a and b must share K and a device, got ", a.sizes(), " on ", dev, ", ",
              b.sizes(), " on ", b.device());
  Tensor bias;
  if (bias_in.has_value()) {
    CHECK_VALUE(bias_in->dim() == 1 && bias_in->size(0) == n && bias_in->device() == dev, "bias must be (", n, ",) on ", dev,
                ", got ", bias_in->sizes(), " on ", bias_in->device());
    bias = bias_in->to(at::kFloat).contiguous();
  }
  if (!THPDtype_Check(dtype.ptr())) throw py::type_error("dtype must be a torch.dtype");
  const at::ScalarType st = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  const int odt = dtype_code(st);
  Tensor out;
  int64_t ldo = std::max<int64_t>(n, 1);
  if (out_in.has_value()) {
    out = *out_in;
    CHECK_VALUE(out.dim() == 2 && out.size(0) == m && out.size(1) == n && out.scalar_type() == st && out.device() == dev &&
                    (n <= 1 || out.stride(1) == 1) && (m <= 1 || out.stride(0) >= n),
                "out must be (", m, ", ", n, ") ", st, " on ", dev, " with contiguous columns");
    if (m > 1) ldo = out.stride(0);
    for (const Tensor* t : {&a, &sa, &b, &sb}) apart(out, *t, "out", "an operand");
    if (bias.defined()) apart(out, bias, "out", "the bias");
  } else {
    out = at::empty_strided({m, n}, {ldo, 1}, a.options().dtype(st));
  }
  const size_t need = lib.matmul_workspace(m, n, k);
  Tensor ws;
  if (need > 0) ws = at::empty_strided({static_cast<int64_t>(need)}, {1}, a.options().dtype(at::kByte));
  lib.status(lib.matmul_blocks(static_cast<const uint8_t*>(ac.data_ptr()), lda, static_cast<const float*>(sa.data_ptr()),
                                   sa.stride(0), sa.stride(1), static_cast<const uint8_t*>(bc.data_ptr()), ldb,
                                   static_cast<const float*>(sb.data_ptr()), sb.stride(0), sb.stride(1), m, n, k,
                                   bias.defined() ? static_cast<const float*>(bias.data_ptr()) : nullptr, out.data_ptr(), odt,
                                   ldo, need ? ws.data_ptr() : nullptr, need, stream_of(a)),
               "vcattn_matmul_blocks");
  if (out_in.has_value()) written(out);
  return out;
}

// ---- packed_attention -------------------------------------------------------------
// What a call needs of a plan.  It owns the records on the device.
struct PackedCall {
  int heads, kv_heads;
  int64_t total_q, total_k, head_dim;
  bool causal;
  vcattn_packed_work work;   // points into `records`
  size_t workspace;
  Tensor records;
};

// Records that a captured graph reads at each replay.  The graph's end may be
// seen on a thread that must not call CUDA, so they are let go by a later call.
struct Ended {
  std::mutex m;
  std::vector<Tensor> records;
  std::atomic<bool> any{false};
};
Ended& ended() {
  static Ended* e = new Ended;   // (graphs may end after this library's statics)
  return *e;
}
void CUDART_CB graph_ended(void* records) {
  Ended& e = ended();
  const std::lock_guard<std::mutex> hold(e.m);
  e.records.push_back(std::move(*static_cast<Tensor*>(records)));
  delete static_cast<Tensor*>(records);
  e.any = true;
}
void drop_ended() {
  Ended& e = ended();
  if (!e.any) return;
  std::vector<Tensor> gone;
  const std::lock_guard<std::mutex> hold(e.m);
  gone.swap(e.records);
  e.any = false;
}

// The records stay what they are until the work on `stream` that reads them is
// done, also if the plan is dropped before: their memory is not handed out
// again while that stream has not passed this call, and a graph that captures
// the call owns them.
void keep_records(const Tensor& records, const c10::cuda::CUDAStream& stream) {
  drop_ended();
  c10::cuda::CUDACachingAllocator::recordStream(records.storage().data_ptr(), stream);
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  cudaGraph_t graph = nullptr;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream.stream(), &status, nullptr, &graph));
  if (status != cudaStreamCaptureStatusActive) return;
  cudaUserObject_t object = nullptr;
  auto held = std::make_unique<Tensor>(records);
  C10_CUDA_CHECK(cudaUserObjectCreate(&object, held.get(), graph_ended, 1, cudaUserObjectNoDestructorSync));
  held.release();
  C10_CUDA_CHECK(cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove));
}

constexpr const char* kPackedCall = "vcattn packed call";

Tensor packed_attention(const Library& lib, const Tensor& q, const Tensor& k, const Tensor& v, const PackedCall& p, std::optional<double> scale,
                        const OptTensor& out_in) {
  refuse_grad("packed_attention", q, k, v, out_in);
  need_cuda(q.is_cuda() && k.is_cuda() && v.is_cuda(), "packed_attention");
  const std::array<int64_t, 4> wq{1, p.heads, p.total_q, p.head_dim}, wk{1, p.kv_heads, p.total_k, p.head_dim};
  CHECK_VALUE(q.sizes() == at::IntArrayRef(wq) && k.sizes() == at::IntArrayRef(wk) && v.sizes() == at::IntArrayRef(wk),
              "the plan needs q ", at::IntArrayRef(wq), " and k, v ", at::IntArrayRef(wk), ", got ", q.sizes(), ", ",
              k.sizes(), ", ", v.sizes());
  const at::ScalarType st = q.scalar_type();
  CHECK_VALUE((st == at::kBFloat16 || st == at::kHalf) && k.scalar_type() == st && v.scalar_type() == st,
              "q, k, v must share bfloat16 or float16, got ", st, ", ", k.scalar_type(), ", ", v.scalar_type());
  const at::Device dev = q.device();
  CHECK_VALUE(k.device() == dev && v.device() == dev && dev == p.records.device(),
              "q, k, v and the plan must be on one device");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(p.head_dim));
  CHECK_VALUE(s > 0.0 && s < 1e30, "scale must be positive and finite, got ", s);
  c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_rows(out_in, q, "out");
  if (out_in.has_value()) {
    in_place_or_apart(out, q, "out", "q");
    apart(out, k, "out", "k");
    apart(out, v, "out", "v");
  }
  const View vq = view(q), vk = view(k), vv = view(v);
  const vcattn_bhnd vo = bhnd(out);
  Tensor ws;
  if (p.workspace > 0) ws = at::empty_strided({static_cast<int64_t>(p.workspace)}, {1}, q.options().dtype(at::kByte));
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(dev.index());
  keep_records(p.records, stream);
  lib.status(lib.attn_packed(&vq.v, &vk.v, &vv.v, dtype_code(st), p.heads, p.kv_heads, static_cast<int>(p.total_q),
                                 static_cast<int>(p.total_k), static_cast<int>(p.head_dim),
                                 &p.work, p.causal ? 1 : 0,
                                 static_cast<float>(s), &vo, p.workspace ? ws.data_ptr() : nullptr, p.workspace,
                                 stream.stream()),
               "vcattn_attn_packed");
  if (out_in.has_value()) written(out);
  return out;
}

Tensor packed_attention_plan(const Library& lib, const Tensor& q, const Tensor& k, const Tensor& v, const py::object& call,
                             std::optional<double> scale, const OptTensor& out) {
  const void* p = PyCapsule_GetPointer(call.ptr(), kPackedCall);
  if (p == nullptr) throw py::error_already_set();
  return packed_attention(lib, q, k, v, *static_cast<const PackedCall*>(p), scale, out);
}

// f with its library.
template <typename R, typename... A> auto with(std::shared_ptr<const Library> lib, R (*f)(const Library&, A...)) {
  return [lib, f](A... a) -> R { return f(*lib, std::forward<A>(a)...); };
}

// The operators of `m`, on these entry points.  (Two copies of the package may
// share this extension's code, so nothing of either is kept outside the module.)
void bind(py::module_ m, const py::dict& d, py::object check) {
  auto lib = std::make_shared<Library>();
  address(d, "vcattn_qk_norm_rope", lib->qk_norm_rope);
  address(d, "vcattn_quantize_blocks", lib->quantize_blocks);
  address(d, "vcattn_matmul_blocks", lib->matmul_blocks);
  address(d, "vcattn_matmul_blocks_workspace_bytes", lib->matmul_workspace);
  address(d, "vcattn_attn_packed", lib->attn_packed);
  lib->check = std::move(check);
  m.def("qk_norm_rope", with(lib, &qk_norm_rope));
  m.def("quantize_blocks", with(lib, &quantize_blocks));
  m.def("matmul_blocks", with(lib, &matmul_blocks));
  m.def("packed_attention", with(lib, &packed_attention_plan));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  // (a capsule: a registered class could not be registered again by a second copy)
  m.def("packed_call", [](int heads, int kv_heads, int64_t total_q, int64_t total_k, int64_t head_dim, bool causal,
                          uintptr_t work, size_t workspace, const Tensor& records) {
    drop_ended();
    return py::capsule(new PackedCall{heads, kv_heads, total_q, total_k, head_dim, causal,
                                      *reinterpret_cast<const vcattn_packed_work*>(work), workspace, records},
                       kPackedCall, [](PyObject* c) { delete static_cast<PackedCall*>(PyCapsule_GetPointer(c, kPackedCall)); });
  });
}
