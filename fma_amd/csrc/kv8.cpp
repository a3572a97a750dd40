// Torch-extension host side of the 8-bit cache and of the norm + rotation
// kernels (kv8.hip). Every call checks what its kernel's grid and indexes
// assume, runs on the current stream of the tensors' device, and takes its
// workspace from the caching allocator, so calls on several streams and
// captured graphs share nothing. A call that does not fit is a ValueError.

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "kv8.h"

namespace {

#define KV8_HIP_CHECK(expr)                                             \
  do {                                                                  \
    hipError_t _e = (expr);                                             \
    /* reported here, not by the next call as well */                   \
    if (_e != hipSuccess) (void)hipGetLastError();                      \
    TORCH_CHECK_VALUE(_e != hipErrorInvalidValue,                       \
                      "sizes beyond one launch, in `" #expr "`");       \
    TORCH_CHECK(_e == hipSuccess, "HIP error — ", hipGetErrorString(_e), \
                " in `" #expr "`");                                     \
  } while (0)

int compute_units(int device) {
  return at::cuda::getDeviceProperties(device)->multiProcessorCount;
}

bool aligned16(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

// [B, T, H, hd], copied if its last dimension is not contiguous.
at::Tensor dense_last(const at::Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 4, name,
                    " must be a GPU tensor [B, T, heads, head_dim]");
  TORCH_CHECK_VALUE(!(x.requires_grad() && at::GradMode::is_enabled()), name,
                    " requires a gradient; there is no backward pass");
  return x.size(3) == 1 || x.stride(3) == 1 ? x : x.contiguous();
}

FmaRows rows_of(const at::Tensor& x) {
  FmaRows r;
  r.p = x.data_ptr();
  r.sb = x.stride(0);
  r.st = x.stride(1);
  r.sh = x.stride(2);
  const int64_t size = x.element_size();
  auto aligned = [&](int64_t stride, int64_t n) {
    return n <= 1 || (stride * size) % 16 == 0;
  };
  r.vec = aligned16(r.p) && x.size(3) % 8 == 0 &&
          aligned(r.sb, x.size(0)) && aligned(r.st, x.size(1)) &&
          aligned(r.sh, x.size(2));
  return r;
}

int type_of(at::ScalarType t) {
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat,
              "bfloat16, float16 or float32 wanted, got ", t);
  return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2;
}

FmaRope rope_of(const c10::optional<at::Tensor>& cos,
                const c10::optional<at::Tensor>& sin,
                const c10::optional<at::Tensor>& qw,
                const c10::optional<at::Tensor>& kw, double eps, bool pairs,
                const at::Tensor& like, int64_t hd) {
  FmaRope r{};
  r.eps = static_cast<float>(eps);
  r.pairs = pairs;
  TORCH_CHECK_VALUE(cos.has_value() == sin.has_value(), "cos and sin go together");
  if (cos.has_value()) {
    const auto &c = *cos, &s = *sin;
    TORCH_CHECK_VALUE(c.device() == like.device() && s.device() == like.device() &&
                    c.scalar_type() == at::kFloat &&
                    s.scalar_type() == at::kFloat && c.dim() == 2 &&
                    c.sizes() == s.sizes() && c.is_contiguous() &&
                    s.is_contiguous(),
                "cos/sin tables must be contiguous fp32 [S, rot/2] beside q");
    TORCH_CHECK_VALUE(c.size(1) >= 1 && 2 * c.size(1) <= hd,
                "the tables rotate more than head_dim");
    TORCH_CHECK_VALUE(c.size(0) >= 1 && c.size(0) <= 0x7fffffff, "bad table length");
    r.cos = c.data_ptr<float>();
    r.sin = s.data_ptr<float>();
    r.half = static_cast<int>(c.size(1));
    r.table = static_cast<int>(c.size(0));
    r.tab_vec = r.half % 4 == 0 && aligned16(r.cos) && aligned16(r.sin);
  }
  auto weight = [&](const c10::optional<at::Tensor>& w) -> const void* {
    if (!w.has_value()) return nullptr;
    TORCH_CHECK_VALUE(!(w->requires_grad() && at::GradMode::is_enabled()),
                      "a norm weight requires a gradient; there is no backward "
                      "pass");
    TORCH_CHECK_VALUE(w->device() == like.device() &&
                    w->scalar_type() == like.scalar_type() &&
                    w->numel() == hd && w->is_contiguous(),
                "norm weights must be contiguous [head_dim] of q's type");
    return w->data_ptr();
  };
  r.qw = weight(qw);
  r.kw = weight(kw);
  r.w_vec = hd % 8 == 0 && aligned16(r.qw) && aligned16(r.kw);
  return r;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& cos,
    const at::Tensor& sin, const c10::optional<at::Tensor>& pos,
    int64_t start, const c10::optional<at::Tensor>& qw,
    const c10::optional<at::Tensor>& kw, double eps, bool pairs) {
  const at::Tensor q = dense_last(q_in, "q"), k = dense_last(k_in, "k");
  const FmaRows qr = rows_of(q), kr = rows_of(k);
  const int64_t B = q.size(0), T = q.size(1), hd = q.size(3);
  TORCH_CHECK_VALUE(k.device() == q.device() && k.scalar_type() == q.scalar_type() &&
                  k.size(0) == B && k.size(1) == T && k.size(3) == hd,
              "k must match q but for the number of heads");
  TORCH_CHECK_VALUE(hd >= 2 && hd <= 256, "head_dim must be 2..256, got ", hd);
  TORCH_CHECK_VALUE(q.size(2) >= 1 && k.size(2) >= 1 && q.size(2) < (1 << 20) &&
                  k.size(2) < (1 << 20) && B < (1 << 30) && T < (1 << 30),
              "bad shape");
  const int type = type_of(q.scalar_type());
  const FmaRope rope = rope_of(cos, sin, qw, kw, eps, pairs, q, hd);
  FmaPos p{};
  p.start = start;
  TORCH_CHECK_VALUE(pos.has_value() || (start >= 0 && start + T <= rope.table),
                    "positions [", start, ", ", start + T,
                    ") lie outside the tables' ", rope.table);
  if (pos.has_value()) {
    const auto& t = *pos;
    TORCH_CHECK_VALUE(t.device() == q.device() && (t.scalar_type() == at::kInt ||
                                             t.scalar_type() == at::kLong),
                "positions must be int32 or int64 beside q");
    TORCH_CHECK_VALUE((t.dim() == 1 && t.size(0) == B) ||
                    (t.dim() == 2 && t.size(0) == B && t.size(1) == T),
                "positions must be [B] or [B, T]");
    if (t.scalar_type() == at::kInt)
      p.p32 = t.data_ptr<int>();
    else
      p.p64 = reinterpret_cast<const long long*>(t.data_ptr<int64_t>());
    p.sb = t.stride(0);
    p.per_token = t.dim() == 2;
    p.st = p.per_token ? t.stride(1) : 0;
  }
  c10::hip::HIPGuard guard(q.device().index());
  auto qo = at::empty({B, T, q.size(2), hd}, q.options());
  auto ko = at::empty({B, T, k.size(2), hd}, q.options());
  auto stream = c10::hip::getCurrentHIPStream(q.device().index());
  KV8_HIP_CHECK(fma_launch_qk_norm_rope(
      qr, kr, qo.data_ptr(), ko.data_ptr(), static_cast<int>(B),
      static_cast<int>(T), static_cast<int>(q.size(2)),
      static_cast<int>(k.size(2)), static_cast<int>(hd), type, rope, p,
      stream.stream()));
  return {qo, ko};
}

// The buffers of one cache, checked once.
class Kv8Buffers {
 public:
  Kv8Buffers(at::Tensor codes, at::Tensor scales, at::Tensor tail,
             int64_t max_seq, int64_t hd, bool fp8)
      : codes_(std::move(codes)), scales_(std::move(scales)),
        tail_(std::move(tail)) {
    TORCH_CHECK_VALUE(codes_.is_cuda() && codes_.scalar_type() == at::kByte &&
                    codes_.dim() == 6 && codes_.is_contiguous(),
                "codes must be uint8 [L, 2, B, kvH, blocks, 32 * width]");
    layers_ = codes_.size(0);
    const int64_t B = codes_.size(2), H = codes_.size(3), n = codes_.size(4);
    const int64_t width = codes_.size(5) / FMA_KV8_BLOCK;
    TORCH_CHECK_VALUE(codes_.size(1) == 2 && layers_ >= 1 && B >= 1 && H >= 1 &&
                    n >= 1 && codes_.size(5) % FMA_KV8_BLOCK == 0,
                "bad shape of codes");
    TORCH_CHECK_VALUE(width == 32 || width == 64 || width == 96 || width == 128 ||
                    width == 192 || width == 256,
                "unsupported width ", width);
    TORCH_CHECK_VALUE(hd >= 1 && hd <= width, "head_dim beyond the width");
    TORCH_CHECK_VALUE(max_seq >= 1 && max_seq <= n * FMA_KV8_BLOCK &&
                    max_seq < (1 << 30),
                "max_seq beyond the blocks");
    TORCH_CHECK_VALUE(B * H < (1 << 30), "too many sequences");
    TORCH_CHECK_VALUE(scales_.device() == codes_.device() &&
                    scales_.scalar_type() == at::kFloat &&
                    scales_.is_contiguous() &&
                    scales_.sizes() == at::IntArrayRef({layers_, 2, B, H, n}),
                "scales must be fp32 [L, 2, B, kvH, blocks]");
    TORCH_CHECK_VALUE(tail_.device() == codes_.device() && tail_.is_contiguous() &&
                    (tail_.scalar_type() == at::kBFloat16 ||
                     tail_.scalar_type() == at::kHalf) &&
                    tail_.sizes() ==
                        at::IntArrayRef({layers_, 2, B, H, 2, codes_.size(5)}),
                "tail must be 16-bit [L, 2, B, kvH, 2, 32 * width]");
    c_.batch = static_cast<int>(B);
    c_.kv_heads = static_cast<int>(H);
    c_.nblk = static_cast<int>(n);
    c_.max_seq = static_cast<int>(max_seq);
    c_.hd = static_cast<int>(hd);
    c_.hdp = static_cast<int>(width);
    c_.fp8 = fp8;
    c_.bf16 = tail_.scalar_type() == at::kBFloat16;
    c_.codes_v = B * H * n * codes_.size(5);
    c_.scales_v = B * H * n;
    c_.tail_v = B * H * 2 * codes_.size(5);
  }

  void append(int64_t layer, const at::Tensor& k, const at::Tensor& v,
              const c10::optional<at::Tensor>& start, int64_t start_i,
              const c10::optional<at::Tensor>& counts) {
    FmaRope none{};
    none.pairs = 1;  // the lighter of the two kernels
    store(layer, nullptr, k, v, none, start, start_i, counts);
  }

  at::Tensor norm_rope_append(
      int64_t layer, const at::Tensor& q, const at::Tensor& k,
      const at::Tensor& v, const at::Tensor& cos, const at::Tensor& sin,
      const c10::optional<at::Tensor>& start, int64_t start_i,
      const c10::optional<at::Tensor>& qw,
      const c10::optional<at::Tensor>& kw,
      const c10::optional<at::Tensor>& counts, double eps, bool pairs) {
    const FmaRope rope = rope_of(cos, sin, qw, kw, eps, pairs, tail_, c_.hd);
    TORCH_CHECK_VALUE(rope.table >= c_.max_seq,
                "the cos/sin tables are shorter than the cache");
    const at::Tensor qd = dense_last(q, "q");
    return store(layer, &qd, k, v, rope, start, start_i, counts);
  }

  std::tuple<at::Tensor, at::Tensor> read(
      int64_t layer, const c10::optional<at::Tensor>& start, int64_t start_i,
      int64_t n, const c10::optional<at::Tensor>& length, int64_t length_i) {
    const FmaKv8Layer c = at_layer(layer);
    TORCH_CHECK_VALUE(n >= 0 && n < (1 << 29) && start_i >= 0 &&
                    start_i < (1 << 30) && length_i >= 0 &&
                    length_i <= c.max_seq,
                "range outside the cache");
    c10::hip::HIPGuard guard(codes_.device().index());
    auto ko = at::empty({c.batch, n, c.kv_heads, c.hd}, tail_.options());
    auto vo = at::empty({c.batch, n, c.kv_heads, c.hd}, tail_.options());
    auto stream = c10::hip::getCurrentHIPStream(codes_.device().index());
    KV8_HIP_CHECK(fma_launch_kv8_read(
        c, per_sequence(start, "start"), static_cast<int>(start_i),
        per_sequence(length, "length"), static_cast<int>(length_i),
        static_cast<int>(n), ko.data_ptr(), vo.data_ptr(), stream.stream()));
    return {ko, vo};
  }

  // Whether a call now would be recorded. The default stream cannot be.
  bool capturing() const {
    hipStream_t stream =
        c10::hip::getCurrentHIPStream(codes_.device().index()).stream();
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (stream != nullptr) KV8_HIP_CHECK(hipStreamIsCapturing(stream, &status));
    return status != hipStreamCaptureStatusNone;
  }

  at::Tensor attention(const at::Tensor& q_in, int64_t layer,
                       const c10::optional<at::Tensor>& start, int64_t start_i,
                       const c10::optional<at::Tensor>& counts, double scale,
                       int64_t held) {
    const FmaKv8Layer c = at_layer(layer);
    at::Tensor q = dense_last(q_in, "q");
    check_new(q, "q");
    FmaRows qr = rows_of(q);
    if (!qr.vec) {
      // the kernel takes rows by 16 bytes
      q = at::constant_pad_nd(q, {0, (8 - c.hd % 8) % 8}).contiguous();
      if (!aligned16(q.data_ptr()) || q.data_ptr() == q_in.data_ptr())
        q = q.clone(at::MemoryFormat::Contiguous);
      qr = rows_of(q);
      TORCH_CHECK(qr.vec, "rows of q are not aligned");
    }
    TORCH_CHECK_VALUE(q.size(2) >= 1 && q.size(2) % c.kv_heads == 0 &&
                    q.size(2) < (1 << 20),
                "query heads must be a multiple of the cache's kv heads");
    FmaKv8Span span = span_of(q.size(1), start, start_i, counts);
    TORCH_CHECK_VALUE(held >= 0 && held <= c.max_seq,
                      "tokens held beyond the cache");
    span.held = static_cast<int>(held);
    c10::hip::HIPGuard guard(q.device().index());
    auto out = at::empty(q_in.sizes(), tail_.options());
    auto stream = c10::hip::getCurrentHIPStream(q.device().index());
    const int q_heads = static_cast<int>(q.size(2));
    const int max_len = span.start != nullptr
                            ? c.max_seq
                            : static_cast<int>(start_i) + span.T;
    const FmaKv8Plan plan = fma_kv8_attn_plan(
        &c, span.T, q_heads, max_len, compute_units(q.device().index()));
    at::Tensor partials;
    float* part = nullptr;
    if (plan.splits > 1) {
      partials = at::empty({q.size(0) * q.size(1) * q_heads, plan.splits,
                            c.hdp + 2},
                           scales_.options());
      part = partials.data_ptr<float>();
    }
    KV8_HIP_CHECK(fma_launch_kv8_attention(c, span, qr, out.data_ptr(),
                                           q_heads, static_cast<float>(scale),
                                           part, plan, stream.stream()));
    return out;
  }

 private:
  FmaKv8Layer at_layer(int64_t layer) const {
    TORCH_CHECK_VALUE(layer >= 0 && layer < layers_, "no layer ", layer);
    FmaKv8Layer c = c_;
    c.codes = codes_.data_ptr<uint8_t>() + layer * 2 * c.codes_v;
    c.scales = scales_.data_ptr<float>() + layer * 2 * c.scales_v;
    c.tail = static_cast<char*>(tail_.data_ptr()) + layer * 4 * c.tail_v;
    return c;
  }

  const int* per_sequence(const c10::optional<at::Tensor>& t,
                          const char* name) const {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK_VALUE(t->device() == codes_.device() &&
                    t->scalar_type() == at::kInt && t->dim() == 1 &&
                    t->size(0) == c_.batch && t->is_contiguous(),
                name, " must be contiguous int32 [B] beside the cache");
    return t->data_ptr<int>();
  }

  void check_new(const at::Tensor& x, const char* name) const {
    TORCH_CHECK_VALUE(x.device() == codes_.device() &&
                    x.scalar_type() == tail_.scalar_type() &&
                    x.size(0) == c_.batch && x.size(3) == c_.hd &&
                    x.size(1) < (1 << 30),
                name, " does not match the cache's device, type, batch or "
                "head_dim");
  }

  FmaKv8Span span_of(int64_t T, const c10::optional<at::Tensor>& start,
                     int64_t start_i,
                     const c10::optional<at::Tensor>& counts) const {
    FmaKv8Span s{};
    s.start = per_sequence(start, "start");
    s.counts = per_sequence(counts, "counts");
    s.T = static_cast<int>(T);
    if (s.start == nullptr) {
      TORCH_CHECK_VALUE(start_i >= 0 && start_i + T <= c_.max_seq,
                  "tokens beyond the cache");
      s.start_i = static_cast<int>(start_i);
    }
    return s;
  }

  at::Tensor store(int64_t layer, const at::Tensor* q, const at::Tensor& k_in,
                   const at::Tensor& v_in, const FmaRope& rope,
                   const c10::optional<at::Tensor>& start, int64_t start_i,
                   const c10::optional<at::Tensor>& counts) {
    const FmaKv8Layer c = at_layer(layer);
    const at::Tensor k = dense_last(k_in, "k"), v = dense_last(v_in, "v");
    const FmaRows kr = rows_of(k), vr = rows_of(v);
    check_new(k, "k");
    check_new(v, "v");
    TORCH_CHECK_VALUE(k.size(2) == c.kv_heads && v.sizes() == k.sizes(),
                "k and v must be [B, T, kvH, head_dim] of the cache");
    const FmaKv8Span span = span_of(k.size(1), start, start_i, counts);
    FmaRows qr{};
    at::Tensor out;
    c10::hip::HIPGuard guard(codes_.device().index());
    int q_heads = 0;
    if (q != nullptr) {
      qr = rows_of(*q);
      check_new(*q, "q");
      TORCH_CHECK_VALUE(q->size(1) == k.size(1) && q->size(2) >= 1 &&
                      q->size(2) % c.kv_heads == 0 && q->size(2) < (1 << 20),
                  "q must be [B, T, a multiple of kvH, head_dim]");
      q_heads = static_cast<int>(q->size(2));
      out = at::empty(q->sizes(), tail_.options());
    }
    auto stream = c10::hip::getCurrentHIPStream(codes_.device().index());
    KV8_HIP_CHECK(fma_launch_kv8_append(
        c, span, qr, kr, vr, q != nullptr ? out.data_ptr() : nullptr, q_heads,
        rope, stream.stream()));
    return out;
  }

  at::Tensor codes_, scales_, tail_;
  int64_t layers_ = 0;
  FmaKv8Layer c_{};
};

}  // namespace

void fma_bind_kv8(pybind11::module_& m) {
  m.def("qk_norm_rope", &qk_norm_rope,
        "Per-head RMSNorm of q and k and the position rotation, one launch",
        py::arg("q"), py::arg("k"), py::arg("cos"), py::arg("sin"),
        py::arg("pos"), py::arg("start"), py::arg("q_norm"),
        py::arg("k_norm"), py::arg("eps"), py::arg("pairs"));
  py::class_<Kv8Buffers>(m, "Kv8Buffers")
      .def(py::init<at::Tensor, at::Tensor, at::Tensor, int64_t, int64_t,
                    bool>(),
           py::arg("codes"), py::arg("scales"), py::arg("tail"),
           py::arg("max_seq"), py::arg("head_dim"), py::arg("fp8"))
      .def("append", &Kv8Buffers::append, py::arg("layer"), py::arg("k"),
           py::arg("v"), py::arg("start"), py::arg("start_i"),
           py::arg("counts"))
      .def("norm_rope_append", &Kv8Buffers::norm_rope_append,
           py::arg("layer"), py::arg("q"), py::arg("k"), py::arg("v"),
           py::arg("cos"), py::arg("sin"), py::arg("start"),
           py::arg("start_i"), py::arg("q_norm"), py::arg("k_norm"),
           py::arg("counts"), py::arg("eps"), py::arg("pairs"))
      .def("capturing", &Kv8Buffers::capturing)
      .def("read", &Kv8Buffers::read, py::arg("layer"), py::arg("start"),
           py::arg("start_i"), py::arg("n"), py::arg("length"),
           py::arg("length_i"))
      .def("attention", &Kv8Buffers::attention, py::arg("q"),
           py::arg("layer"), py::arg("start"), py::arg("start_i"),
           py::arg("counts"), py::arg("scale"), py::arg("held"));
}
