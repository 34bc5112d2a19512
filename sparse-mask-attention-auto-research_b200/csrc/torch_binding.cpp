// PyTorch side of the operators on queries and keys of different lengths
// (python/cross_attention.py): argument checks, workspaces, the choice between
// the entry points of libsma.so, and the autograd node.
//
// These calls are as short as a generated token's, where the host bounds them:
// the same steps in Python cost 12.6 us a call against 6 us here (one token
// over 128 keys, whose kernel takes 4 us), and a training pass through a
// Python autograd node 145 us against 76 us.
//
// libsma.so itself stays free of torch: bind() hands its entry points over.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>

#include "sma_capi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&sma_rows_attn_fwd) rows = nullptr;
  decltype(&sma_cross_attn_fwd) cross = nullptr;
  decltype(&sma_prefix_attn_fwd) prefix = nullptr;
  decltype(&sma_cross_attn_bwd) cross_bwd = nullptr;
  decltype(&sma_cross_attn_bwd_f32_table) cross_bwd_f32_table = nullptr;
  decltype(&sma_cross_attn_bwd_scratch) cross_bwd_scratch = nullptr;
  decltype(&sma_last_error) last_error = nullptr;
} api;

// A non-zero status of an entry point; SmaError in Python.
struct Status : std::runtime_error {
  Status(int c, const char* text)
      : std::runtime_error("[sma status " + std::to_string(c) + "] " + text), code(c), message(text) {}
  int code;
  std::string message;
};

void check(int code) {
  if (code != SMA_OK) throw Status(code, api.last_error());
}

// With gradients: 64-row steps of the queries of all heads that share a key head.
constexpr int64_t kMaxSteps = 2048;

// Backward mode, or forward mode (which the node refuses).
bool needs_grad(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined()) return true;
  return false;
}

void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "attention requires CUDA tensors (no CPU fallback)");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q/k/v must be on the same device");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "q must be [B, H, Nq, D], k and v [B, Hkv, Nk, D]");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "q/k/v must have the same dtype");
  const auto t = q.scalar_type();
  TORCH_CHECK(t == at::kHalf || t == at::kBFloat16 || t == at::kFloat, "Unsupported dtype, need BF16, FP16 or FP32");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3), "q/k/v must agree in batch and head dim");
  TORCH_CHECK(q.size(3) == 64 || q.size(3) == 128, "head dim must be 64 or 128");
  const int64_t H = q.size(1), Hkv = k.size(1);
  TORCH_CHECK(H == 0 || (Hkv > 0 && H % Hkv == 0), "the key heads must divide the query heads");
}

void check_mask(const Tensor& mask, const Tensor& q, const Tensor& k) {
  TORCH_CHECK(mask.device() == q.device(), "mask must be on the same device as q");
  TORCH_CHECK(mask.scalar_type() == at::kBool, "mask must be a bool tensor");
  bool ok = mask.dim() == 4 && mask.size(3) == k.size(2);
  for (int i = 0; ok && i < 3; ++i) ok = mask.size(i) == 1 || mask.size(i) == q.size(i);
  TORCH_CHECK(ok, "mask must broadcast to [", q.size(0), ", ", q.size(1), ", ", q.size(2), ", ", k.size(2),
              "] along its first three axes, got ", mask.sizes());
}

double scale_of(std::optional<double> scale, int64_t D) {
  if (!scale.has_value()) return 1.0 / std::sqrt(static_cast<double>(D));
  TORCH_CHECK(*scale > 0.0 && std::isfinite(*scale), "scale must be finite and > 0");
  return *scale;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// `t`, or a contiguous copy of it where the kernels cannot step along its
// strides (last axis contiguous, the others positive multiples of 16 bytes, a
// 16-byte aligned base).
Tensor strided(const Tensor& t) {
  const bool aligned = aligned16(t.const_data_ptr());
  if (t.is_contiguous()) return aligned ? t : t.clone(at::MemoryFormat::Contiguous);
  const int64_t last = t.dim() - 1;
  bool ok = aligned && t.stride(last) == 1;
  for (int64_t i = 0; ok && i < last; ++i) ok = t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0);
  return ok ? t : t.contiguous();
}

Tensor empty(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

// A bool mask [B or 1, H or 1, Nq or 1, Nk] with a contiguous last axis, and
// its strides along the others (0 where it is broadcast).
struct Mask {
  Tensor t;
  std::array<int64_t, 3> stride{};
  bool on() const { return t.defined(); }
};
Mask mask_of(const std::optional<Tensor>& mask) {
  Mask m;
  if (!mask.has_value()) return m;
  m.t = mask->size(3) > 1 && mask->stride(3) != 1 ? mask->contiguous() : *mask;
  for (int i = 0; i < 3; ++i) m.stride[i] = m.t.size(i) == 1 ? 0 : m.t.stride(i);
  return m;
}

// A bias table as the kernels read it, of q's type.
Tensor table_of(const std::optional<Tensor>& table, const Tensor& q) {
  return table.has_value() ? table->to(q.scalar_type()).contiguous() : Tensor();
}

// A relative position bias; its table and offsets are passed beside it.
struct Bias {
  bool on = false, two_sided = false;
  int32_t side = 0;
  int64_t offset = 0;
  std::array<int32_t, SMA_MAX_BIAS_SIDE> starts{};
};

sma_attn_args args_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, double scale) {
  sma_attn_args a{};
  a.dtype = q.scalar_type() == at::kHalf ? SMA_DTYPE_FP16 : SMA_DTYPE_BF16;
  a.scale = static_cast<float>(scale);
  a.B = q.size(0), a.H = q.size(1), a.Hkv = k.size(1), a.Nq = q.size(2), a.Nk = k.size(2), a.D = q.size(3);
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr();
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q.stride(i), a.k_stride[i] = k.stride(i), a.v_stride[i] = v.stride(i);
  a.out = out.data_ptr();
  return a;
}

void set_bias(sma_attn_args* a, const Bias& bias, const Tensor& table, const Tensor& offsets) {
  if (!bias.on) return;
  a->bias_table = table.const_data_ptr();
  a->bias_starts = bias.starts.data();
  a->bias_offsets = offsets.defined() ? offsets.const_data_ptr<int32_t>() : nullptr;
  a->bias_offset = bias.offset;
  a->bias_side = bias.side;
  a->bias_two_sided = bias.two_sided ? 1 : 0;
}

// The buffer that a forward on 128-row tiles fills for itself and its backward:
// byte offsets (0: none; the first 16 bytes are not used) and its size.
struct Layout {
  int64_t words = 0, distance = 0, lse = 0, out_lo = 0, bytes = 16;
};
Layout layout_of(const Tensor& q, const Tensor& k, bool masked, const std::array<int64_t, 3>& mask_stride,
                 const Bias& bias, bool training) {
  const auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
  Layout l;
  if (masked) {
    l.words = l.bytes;
    int64_t rows = 1, tiles = 1;
    for (int i = 0; i < 3; ++i) {
      if (mask_stride[i] == 0) continue;
      const int64_t n = q.size(i);
      rows *= n;
      tiles *= i == 2 ? (n + 127) / 128 : n;
    }
    const int64_t Nk = k.size(2), W = (Nk + 127) / 128 * 4;
    l.bytes += (rows + tiles) * W * 4 + up(tiles * ((Nk + 2047) / 2048) * 4);
  }
  if (bias.on) {
    l.distance = l.bytes;
    l.bytes += q.size(1) * 4 * SMA_BIAS_DISTANCE_LEN(bias.starts[bias.side - 1], bias.two_sided);
  }
  if (training) {
    l.lse = l.bytes;
    l.bytes += up(q.size(0) * q.size(1) * q.size(2) * 4);
    l.out_lo = l.bytes;
    l.bytes += q.numel() * 2;
  }
  return l;
}

void set_saved(sma_attn_args* a, const Layout& l, const Tensor& saved) {
  if (!saved.defined()) return;
  uint8_t* base = static_cast<uint8_t*>(saved.data_ptr());
  if (l.words) a->words = base + l.words;
  if (l.distance) a->bias_distance = reinterpret_cast<float*>(base + l.distance);
  if (l.lse) a->lse = reinterpret_cast<float*>(base + l.lse);
  if (l.out_lo) a->out_lo = base + l.out_lo;
}

// Whether the streaming kernel is taken (16 rows of a key head at a time, the
// keys read again for every 16) instead of the 128-row tiles.
//
// With no mask, or one that all rows of a key head share, and R rows per key
// head in T tiles of 128, the first takes (measured on a B200) about 6 us +
// B Hkv Nk D ceil(R / 16) * 0.57e-6 us, the second (which also packs the
// mask) 15 us + B Hkv Nk D T * 0.9e-6 us (D = 64) or 0.77e-6 us (D = 128).
// For instance B8 Hkv8 Nk1000 D64: 12.1 against 20.3 us at 64 rows, 19.9 at
// 96, 21.9 at 112; B16 H12 Nk1500 D128: 31 against 48 us at 16 rows, 58
// against 48 at 24.  Masks of the rows' own and a bias cost the first more:
// B16 H12 Nk500 D64 with a mask 19.4 against 20.9 us at 16 rows, 35.5 against
// 21.0 at 32, so there it is taken for one tile of 16 rows only.
bool few_rows(const Tensor& q, const Tensor& k, const Mask& mask, const Bias& bias) {
  const int64_t B = q.size(0), H = q.size(1), Nq = q.size(2), D = q.size(3), Hkv = k.size(1), Nk = k.size(2);
  if (Nk > SMA_MAX_SEQ_LEN) return true;
  const int64_t rows = H / std::max<int64_t>(Hkv, 1) * Nq;
  if (rows <= 16 || rows > 128) return rows <= 16;
  // A mask that all rows of a key head share may still be an expanded view.
  const bool own_rows = mask.on() && ((Nq > 1 && mask.stride[2] != 0) || (H > Hkv && mask.stride[1] != 0));
  if (bias.on || own_rows) return false;
  const double tiles = static_cast<double>((rows + 15) / 16);
  return static_cast<double>(B * Hkv * Nk * D) * ((D == 64 ? 0.6 : 0.75) * tiles - 1.0) <= 12e6;
}

void* current_stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// sma_cross_attn_fwd: writes `out`; returns the buffer of layout `l` that it filled.
Tensor tiles_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, double scale,
                     const Mask& mask, const Bias& bias, const Tensor& table, const Tensor& offsets, const Layout& l) {
  Tensor saved;
  if (l.bytes > 16) saved = at::empty({l.bytes}, q.options().dtype(at::kByte));
  sma_attn_args a = args_of(q, k, v, out, scale);
  if (mask.on()) {
    a.mask = mask.t.const_data_ptr();
    for (int i = 0; i < 3; ++i) a.mask_stride[i] = mask.stride[i];
  }
  set_bias(&a, bias, table, offsets);
  set_saved(&a, l, saved);
  check(api.cross(&a, current_stream(q)));
  return saved;
}

// What a node keeps beside its tensors.
struct Plan : torch::CustomClassHolder {
  double scale = 0.0;
  Bias bias;
  Layout layout;
  std::array<int64_t, 3> mask_stride{};
  bool table_f32 = false;  // the caller's table, and so its gradient
};

// Autograd node of cross_attention (no table) and relative_bias_attention.
struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_,
                        const std::optional<Tensor>& table_, const std::optional<Tensor>& mask_,
                        const std::optional<Tensor>& offsets_, double scale, const Bias& bias) {
    const Tensor q = strided(q_), k = strided(k_), v = strided(v_);
    const Tensor table = table_of(table_, q), offsets = offsets_.value_or(Tensor());
    const Mask mask = mask_of(mask_);
    auto plan = c10::make_intrusive<Plan>();
    plan->scale = scale;
    plan->bias = bias;
    plan->layout = layout_of(q, k, mask.on(), mask.stride, bias, true);
    plan->mask_stride = mask.stride;
    plan->table_f32 = table_.has_value() && table_->scalar_type() == at::kFloat;
    const Tensor out = empty(q);
    const Tensor saved = tiles_forward(q, k, v, out, scale, mask, bias, table, offsets, plan->layout);
    ctx->save_for_backward({q, k, v, out, saved, table, offsets});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(std::move(plan));
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto kept = ctx->get_saved_variables();
    const Tensor &q = kept[0], &k = kept[1], &v = kept[2], &out = kept[3], &saved = kept[4], &table = kept[5];
    const auto capsule = ctx->saved_data["plan"].toCapsule();
    const Plan& plan = *static_cast<const Plan*>(capsule.get());
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor dout = grads[0].contiguous();
    if (!aligned16(dout.const_data_ptr())) dout = dout.clone();
    Tensor dq = empty(q), dk = empty(k), dv = empty(k), dtable;
    if (table.defined()) dtable = at::empty(table.sizes(), plan.table_f32 ? table.options().dtype(at::kFloat) : table.options());
    if (q.numel() == 0 || k.numel() == 0) {
      for (Tensor* t : {&dq, &dk, &dv, &dtable})
        if (t->defined()) t->zero_();
    } else {
      sma_attn_args a = args_of(q, k, v, out, plan.scale);
      for (int i = 0; i < 3; ++i) a.mask_stride[i] = plan.mask_stride[i];
      set_bias(&a, plan.bias, table, kept[6]);
      set_saved(&a, plan.layout, saved);
      const int64_t floats = api.cross_bwd_scratch(&a);
      TORCH_CHECK(floats >= 0, "backward: unsupported arguments");
      const Tensor scratch = at::empty({floats}, q.options().dtype(at::kFloat));
      if (plan.table_f32) {
        check(api.cross_bwd_f32_table(&a, dout.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                      dtable.data_ptr<float>(), scratch.data_ptr<float>(), current_stream(q)));
      } else {
        check(api.cross_bwd(&a, dout.const_data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                            dtable.defined() ? dtable.data_ptr() : nullptr, scratch.data_ptr<float>(),
                            current_stream(q)));
      }
    }
    variable_list out_grads = {dq, dk, dv, dtable};
    // Differentiable once: what is built on these gradients says so when it is
    // differentiated.  They depend on q, k, v and the table even where the
    // incoming gradient is a constant, so create_graph alone decides.
    if (at::GradMode::is_enabled()) {
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "the gradients of this attention cannot be differentiated again", static_cast<int64_t>(out_grads.size()));
      for (Tensor& t : out_grads)
        if (t.defined()) t.set_requires_grad(true);
      out_grads = (*error)(std::move(out_grads));
    }
    out_grads.resize(8);  // mask, offsets, scale, bias
    return out_grads;
  }
};

// out [B, H, Nq, D] of checked fp16 / bf16 inputs.  `table` is the caller's: of
// q's type or FP32.
Tensor attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const std::optional<Tensor>& table,
                 const std::optional<Tensor>& mask_, const std::optional<Tensor>& offsets, double scale,
                 const Bias& bias) {
  const c10::cuda::CUDAGuard guard(q_.device());
  if (needs_grad({&q_, &k_, &v_}) || (table.has_value() && needs_grad({&*table}))) {
    const int64_t steps = q_.size(1) / std::max<int64_t>(k_.size(1), 1) * ((q_.size(2) + 63) / 64);
    TORCH_CHECK(k_.size(2) <= SMA_MAX_SEQ_LEN, "with gradients at most ", SMA_MAX_SEQ_LEN, " keys are supported");
    TORCH_CHECK(steps <= kMaxSteps, "with gradients at most ", kMaxSteps,
                " steps of 64 queries may share a key head");
    return CrossAttention::apply(q_, k_, v_, table, mask_, offsets, scale, bias);
  }
  const Tensor q = strided(q_), k = strided(k_), v = strided(v_);
  const Mask mask = mask_of(mask_);
  const Tensor out = empty(q);
  const Tensor tab = table_of(table, q), off = offsets.value_or(Tensor());
  if (few_rows(q, k, mask, bias)) {
    sma_attn_args a = args_of(q, k, v, out, scale);
    if (mask.on()) {
      a.mask = mask.t.const_data_ptr();
      for (int i = 0; i < 3; ++i) a.mask_stride[i] = mask.stride[i];
    }
    set_bias(&a, bias, tab, off);
    check(api.rows(&a, current_stream(q)));
  } else {
    tiles_forward(q, k, v, out, scale, mask, bias, tab, off,
                  layout_of(q, k, mask.on(), mask.stride, bias, false));
  }
  return out;
}

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask,
                       std::optional<double> scale_) {
  check_qkv(q, k, v);
  if (mask.has_value()) check_mask(*mask, q, k);
  const double scale = scale_of(scale_, q.size(3));
  const Bias none;
  if (q.scalar_type() != at::kFloat) return attention(q, k, v, std::nullopt, mask, std::nullopt, scale, none);
  return attention(q.to(at::kBFloat16), k.to(at::kBFloat16), v.to(at::kBFloat16), std::nullopt, mask, std::nullopt,
                   scale, none)
      .to(at::kFloat);
}

// `starts`: host address of one side's `side` bucket starts (copied here).
Tensor relative_bias_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                               const std::optional<Tensor>& mask, uintptr_t starts, int64_t side, bool two_sided,
                               int64_t offset, const std::optional<Tensor>& offsets_, std::optional<double> scale_) {
  check_qkv(q, k, v);
  if (mask.has_value()) check_mask(*mask, q, k);
  TORCH_CHECK(table.device() == q.device(), "table must be on the same device as q");
  TORCH_CHECK(table.dim() == 2 && table.size(1) == q.size(1), "table must be [num_buckets, H]");
  TORCH_CHECK(table.scalar_type() == q.scalar_type() || table.scalar_type() == at::kFloat,
              "table must have the dtype of q or be FP32");
  std::optional<Tensor> offsets = offsets_;
  if (offsets.has_value()) {
    TORCH_CHECK(offsets->device() == q.device() && offsets->scalar_type() == at::kInt && offsets->dim() == 1 &&
                    offsets->size(0) == q.size(0),
                "query_offset must be an int or an int32 tensor [B] on the device of q");
    offsets = offsets->contiguous();
  }
  const double scale = scale_of(scale_, q.size(3));
  TORCH_CHECK(side >= 1 && side <= SMA_MAX_BIAS_SIDE, "1 to ", SMA_MAX_BIAS_SIDE, " buckets per side are supported");
  Bias bias;
  bias.on = true;
  bias.two_sided = two_sided;
  bias.side = static_cast<int32_t>(side);
  bias.offset = offset;
  std::copy_n(reinterpret_cast<const int32_t*>(starts), side, bias.starts.begin());
  const bool fp32 = q.scalar_type() == at::kFloat;
  if (!fp32) return attention(q, k, v, table, mask, offsets, scale, bias);
  return attention(q.to(at::kBFloat16), k.to(at::kBFloat16), v.to(at::kBFloat16), table, mask, offsets, scale, bias)
      .to(at::kFloat);
}

Tensor shared_prefix_attention(const Tensor& q_, const Tensor& kp_, const Tensor& vp_, const Tensor& k_,
                               const Tensor& v_, const std::optional<Tensor>& lengths_,
                               std::optional<double> scale_) {
  check_qkv(q_, k_, v_);
  TORCH_CHECK(kp_.is_cuda() && vp_.is_cuda(), "attention requires CUDA tensors (no CPU fallback)");
  TORCH_CHECK(kp_.device() == q_.device() && vp_.device() == q_.device(),
              "the prefix must be on the same device as q");
  TORCH_CHECK(kp_.scalar_type() == q_.scalar_type() && vp_.scalar_type() == q_.scalar_type(),
              "the prefix must have the dtype of q");
  TORCH_CHECK(kp_.dim() == 3 && kp_.sizes() == vp_.sizes() && kp_.size(0) == k_.size(1) && kp_.size(2) == q_.size(3),
              "k_prefix and v_prefix must be [Hkv, P, D]");
  TORCH_CHECK(!needs_grad({&q_, &kp_, &vp_, &k_, &v_}),
              "shared_prefix_attention is forward only (use torch.no_grad())");
  const int64_t B = q_.size(0), T = q_.size(2), S = k_.size(2);
  const c10::cuda::CUDAGuard guard(q_.device());
  Tensor lengths;
  if (lengths_.has_value()) {
    TORCH_CHECK(lengths_->device() == q_.device() && lengths_->scalar_type() == at::kInt && lengths_->dim() == 1 &&
                    lengths_->size(0) == B,
                "lengths must be an int32 tensor [B] on the device of q");
    lengths = lengths_->contiguous();
  } else if (T > 1) {
    lengths = at::full({B}, S, q_.options().dtype(at::kInt));
  }
  const double scale = scale_of(scale_, q_.size(3));
  const bool fp32 = q_.scalar_type() == at::kFloat;
  const auto in = [&](const Tensor& t) { return strided(fp32 ? t.to(at::kBFloat16) : t); };
  const Tensor q = in(q_), kp = in(kp_), vp = in(vp_), k = in(k_), v = in(v_);
  const Tensor out = empty(q);
  sma_attn_args a = args_of(q, k, v, out, scale);
  if (lengths.defined()) a.lengths = lengths.const_data_ptr<int32_t>();
  a.P = kp.size(1);
  if (a.P > 0) {
    a.k_prefix = kp.const_data_ptr(), a.v_prefix = vp.const_data_ptr();
    for (int i = 0; i < 2; ++i) a.kp_stride[i] = kp.stride(i), a.vp_stride[i] = vp.stride(i);
  }
  check((a.P == 0 || S > SMA_MAX_SEQ_LEN ? api.rows : api.prefix)(&a, current_stream(q)));
  return fp32 ? out.to(at::kFloat) : out;
}

// Addresses of libsma.so's entry points by name.
void bind(const py::dict& at, py::object sma_error) {
  const auto get = [&](const char* name) { return at[name].cast<uintptr_t>(); };
  api.rows = reinterpret_cast<decltype(api.rows)>(get("sma_rows_attn_fwd"));
  api.cross = reinterpret_cast<decltype(api.cross)>(get("sma_cross_attn_fwd"));
  api.prefix = reinterpret_cast<decltype(api.prefix)>(get("sma_prefix_attn_fwd"));
  api.cross_bwd = reinterpret_cast<decltype(api.cross_bwd)>(get("sma_cross_attn_bwd"));
  api.cross_bwd_f32_table = reinterpret_cast<decltype(api.cross_bwd_f32_table)>(get("sma_cross_attn_bwd_f32_table"));
  api.cross_bwd_scratch = reinterpret_cast<decltype(api.cross_bwd_scratch)>(get("sma_cross_attn_bwd_scratch"));
  api.last_error = reinterpret_cast<decltype(api.last_error)>(get("sma_last_error"));
  static py::object error;
  error = std::move(sma_error);
  error.inc_ref();  // outlives the interpreter's shutdown
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Status& s) {
      const py::object e = error(s.code, s.message);
      PyErr_SetObject(error.ptr(), e.ptr());
    } catch (const py::error_already_set&) {
      throw;
    } catch (const py::builtin_exception&) {
      throw;
    } catch (const std::exception&) {  // a failed check, no memory left, ...: as torch raises them
      torch::translate_exception_to_python(std::current_exception());
    }
  });
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("bind", &bind);
  m.def("cross_attention", &cross_attention, no_gil);
  m.def("relative_bias_attention", &relative_bias_attention, no_gil);
  m.def("shared_prefix_attention", &shared_prefix_attention, no_gil);
}
