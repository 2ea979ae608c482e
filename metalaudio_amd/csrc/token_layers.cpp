// Argument checks and launch planning of the token layers; the arithmetic is in k_rmsnorm.hip,
// k_linear_e4m3.hip, k_rotary.hip, k_window.hip and k_window_step.hip.
#include "token_layers.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "token_ops.hpp"

namespace mnn {

namespace {

LaunchCtx ctx(Stream& s) { return LaunchCtx{s.dev, s.s}; }

bool is_float(const Tensor& t) { return t.dtype == MNN_F32 || t.dtype == MNN_BF16; }

// Whether two tensors hold the same memory (tensors are whole allocations).
bool same(const Tensor* a, const Tensor* b) { return a && b && a->data && a->data == b->data; }

// Device memory that grows without freeing what it had: a graph captured before a larger call still
// names the earlier block. Each growth is at least half as much again, so that the blocks together
// stay below three times the last.
class Scratch {
 public:
  void* get(size_t n) {
    if (n <= size_) return blocks_.back()->ptr;
    auto b = std::make_unique<DevBuf>();
    const size_t want = std::max(n, size_ + size_ / 2);
    b->reserve(want);
    blocks_.push_back(std::move(b));
    size_ = want;
    return blocks_.back()->ptr;
  }

 private:
  std::vector<std::unique_ptr<DevBuf>> blocks_;
  size_t size_ = 0;
};

// Layers without a one-input forward.
class ManyInputLayer : public Layer {
 public:
  using Layer::Layer;
  Shape infer_output(const Shape& in) const override { return in; }
  void forward(const Tensor&, Tensor&, Stream&) override {
    fail(MNN_ERR_INVALID_CONFIGURATION, std::string(kind()) + " has no one-input forward");
  }
};

template <class T>
T& as(Layer* l, const char* what) {
  T* t = dynamic_cast<T*>(l);
  MNN_REQUIRE(t, MNN_ERR_INVALID_ARGUMENT, what << ": the layer is a " << l->kind());
  return *t;
}

// [S, W] / [B, S, W] with W = n * hd
void split_heads(const char* what, const Shape& s, int64_t hd, int64_t& B, int64_t& S, int64_t& n) {
  MNN_REQUIRE((s.size() == 2 || s.size() == 3) && s.back() > 0 && s.back() % hd == 0,
              MNN_ERR_SHAPE_MISMATCH, what << ": expected [S, heads * " << hd << "] or [B, S, heads * "
                                           << hd << "], got " << shape_str(s));
  B = s.size() == 3 ? s[0] : 1;
  S = s[s.size() - 2];
  n = s.back() / hd;
}

// ------------------------------------------------------------------ RMSNorm
class RMSNormLayer : public Layer {
 public:
  RMSNormLayer(Device* d, int features, float eps) : Layer(d), F_(features), eps_(eps) {
    MNN_REQUIRE(features > 0 && features <= (1 << 30), MNN_ERR_INVALID_CONFIGURATION,
                "RMSNorm: featureSize must be 1..2^30");
    MNN_REQUIRE(std::isfinite(eps) && eps >= 0.f, MNN_ERR_INVALID_CONFIGURATION,
                "RMSNorm: epsilon must be finite and not negative");
    w_ = &add_param("weight", features, 1.f);
    aliases_["gamma"] = "weight";
  }
  const char* kind() const override { return "RMSNorm"; }
  Shape input_shape() const override { return {F_}; }
  Shape output_shape() const override { return {F_}; }
  Shape infer_output(const Shape& in) const override {
    MNN_REQUIRE(!in.empty() && in.back() == F_, MNN_ERR_SHAPE_MISMATCH,
                "RMSNorm: expected last dimension " << F_ << ", got " << shape_str(in));
    return in;
  }
  bool accepts_bf16() const override { return true; }
  void forward(const Tensor& in, Tensor& out, Stream& s) override {
    check_out(out, infer_output(in.shape));
    run(in, nullptr, nullptr, out, nullptr, s);
  }
  void run(const Tensor& in, const Tensor* res, Tensor* sum, Tensor& out, Tensor* scales, Stream& s) {
    infer_output(in.shape);
    const int64_t rows = in.count() / F_;
    MNN_REQUIRE(is_float(in) && (!res || res->dtype == in.dtype) && (!sum || sum->dtype == in.dtype),
                MNN_ERR_INVALID_ARGUMENT,
                "RMSNorm: input, residual and sum must all be f32 or all bf16");
    MNN_REQUIRE(is_float(out) || out.dtype == MNN_E4M3, MNN_ERR_INVALID_ARGUMENT,
                "RMSNorm: output must be f32, bf16 or e4m3");
    MNN_REQUIRE((out.dtype == MNN_E4M3) == (scales != nullptr), MNN_ERR_INVALID_ARGUMENT,
                "RMSNorm: scales go with an e4m3 output");
    MNN_REQUIRE(!scales || scales->dtype == MNN_F32, MNN_ERR_INVALID_ARGUMENT,
                "RMSNorm: scales must be f32");
    for (const Tensor* t : {res, (const Tensor*)sum, (const Tensor*)&out})
      MNN_REQUIRE(!t || t->count() == in.count(), MNN_ERR_BUFFER_SIZE_MISMATCH,
                  "RMSNorm: " << shape_str(t->shape) << " beside an input of " << shape_str(in.shape));
    MNN_REQUIRE(!scales || scales->count() == rows, MNN_ERR_BUFFER_SIZE_MISMATCH,
                "RMSNorm: " << scales->count() << " scales for " << rows << " rows");
    MNN_REQUIRE(!same(sum, &out), MNN_ERR_INVALID_ARGUMENT, "RMSNorm: sum and output are one tensor");
    for (const Tensor* t : {&in, res, (const Tensor*)sum, (const Tensor*)&out})
      MNN_REQUIRE(!same(scales, t), MNN_ERR_INVALID_ARGUMENT,
                  "RMSNorm: the scales are another argument too");
    MNN_REQUIRE(out.dtype == in.dtype || !(same(&in, &out) || same(res, &out)),
                MNN_ERR_INVALID_ARGUMENT, "RMSNorm: in place only with one type");
    k::RmsNormArgs a;
    a.x = in.data;
    a.r = res ? res->data : nullptr;
    a.sum = sum ? sum->data : nullptr;
    a.in = in.dtype;
    a.w = w_->ptr();
    a.y = out.data;
    a.out = out.dtype;
    a.scales = scales ? scales->f32() : nullptr;
    a.rows = rows;
    a.F = F_;
    a.ldy = F_;
    a.eps = eps_;
    k::rmsnorm(ctx(s), a);
  }

 private:
  int F_;
  float eps_;
  Param* w_;
};

// ------------------------------------------------------------------ Linear in 8 bits
// Weights are kept as e4m3 rows, padded with zeros to a multiple of the product's depth step, beside one
// scale a row; no fp32 copy stays on the device.
class LinearE4m3Layer : public Layer {
 public:
  LinearE4m3Layer(Device* d, int in, int out, bool bias, int act, float alpha)
      : Layer(d), in_(in), out_(out), act_(act), alpha_(alpha) {
    MNN_REQUIRE(in > 0 && out > 0, MNN_ERR_INVALID_CONFIGURATION, "Linear: sizes must be > 0");
    MNN_REQUIRE(in <= (1 << 20) && out <= (1 << 24), MNN_ERR_INVALID_CONFIGURATION,
                "Linear: more than 2^20 inputs or 2^24 outputs in 8 bits");
    MNN_REQUIRE(std::isfinite(alpha), MNN_ERR_INVALID_CONFIGURATION,
                "FusedLinear: leakyReluAlpha must be finite");
    if (bias) b_ = &add_param("bias", out);
    kp_ = (in + 127) / 128 * 128;
    dev_->make_current();
    wq_.reserve((size_t)out * kp_);
    ws_.reserve(sizeof(float) * out);
    HIP_CHECK(hipMemset(wq_.ptr, 0, (size_t)out * kp_));  // zero until loaded
    HIP_CHECK(hipMemset(ws_.ptr, 0, sizeof(float) * out));
    HIP_CHECK(hipStreamSynchronize(nullptr));  // streams that do not wait for the null stream read them
  }
  const char* kind() const override { return "Linear"; }
  Shape input_shape() const override { return {in_}; }
  Shape output_shape() const override { return {out_}; }
  Shape infer_output(const Shape& in) const override {
    MNN_REQUIRE(!in.empty() && in.back() == in_, MNN_ERR_SHAPE_MISMATCH,
                "Linear: expected last dimension " << in_ << ", got " << shape_str(in));
    Shape o = in;
    o.back() = out_;
    return o;
  }
  bool accepts_bf16() const override { return true; }
  void load(const std::string& name, const float* data, size_t n) override {
    if (name != "weight") return Layer::load(name, data, n);
    MNN_REQUIRE(n == (size_t)in_ * out_, MNN_ERR_BUFFER_SIZE_MISMATCH,
                "Linear parameter 'weight': expected " << (size_t)in_ * out_ << " values, got " << n);
    MNN_REQUIRE(data, MNN_ERR_INVALID_ARGUMENT, "null data");
    uint32_t bad = 0;  // all values at once, a loop that the compiler can vectorise
    for (size_t i = 0; i < n; ++i) {
      uint32_t u;
      std::memcpy(&u, data + i, 4);
      bad |= (uint32_t)((u & 0x7f800000u) == 0x7f800000u);
    }
    for (size_t i = 0; bad && i < n; ++i) {
      MNN_REQUIRE(!std::isnan(data[i]), MNN_ERR_INVALID_CONFIGURATION,
                  name << " contain NaN values - model file may be corrupted");
      MNN_REQUIRE(!std::isinf(data[i]), MNN_ERR_INVALID_CONFIGURATION,
                  name << " contain Inf values - possible exploding gradients during training");
    }
    set_weights(data);
  }
  void forward(const Tensor& in, Tensor& out, Stream& s) override {
    check_out(out, infer_output(in.shape));
    run(in, nullptr, nullptr, out, s);
  }
  void run(const Tensor& in, const Tensor* scales, const Tensor* res, Tensor& out, Stream& s) {
    const int64_t rows = numel(infer_output(in.shape)) / out_;
    MNN_REQUIRE((in.dtype == MNN_E4M3 && scales) || (is_float(in) && !scales),
                MNN_ERR_INVALID_ARGUMENT,
                "Linear: input must be e4m3 with scales, or f32 or bf16 without");
    MNN_REQUIRE(is_float(out) && (!res || res->dtype == out.dtype), MNN_ERR_INVALID_ARGUMENT,
                "Linear: output must be f32 or bf16 and the residual of the same type");
    MNN_REQUIRE(!scales || scales->dtype == MNN_F32, MNN_ERR_INVALID_ARGUMENT,
                "Linear: scales must be f32");
    for (const Tensor* t : {res, (const Tensor*)&out})
      MNN_REQUIRE(!t || t->count() == rows * out_, MNN_ERR_BUFFER_SIZE_MISMATCH,
                  "Linear: " << shape_str(t->shape) << " for " << rows << " rows of " << out_);
    MNN_REQUIRE(!scales || scales->count() == rows, MNN_ERR_BUFFER_SIZE_MISMATCH,
                "Linear: " << scales->count() << " scales for " << rows << " rows");
    MNN_REQUIRE(!same(&in, &out) && !same(scales, &out), MNN_ERR_INVALID_ARGUMENT,
                "Linear: output is the input or its scales");
    if (rows == 0) return;
    k::LinearE4m3Args g;
    g.x = static_cast<const uint8_t*>(in.data);
    g.xs = scales ? scales->f32() : nullptr;
    if (!scales) {  // rows rounded to 8 bits first, their scales behind them
      const size_t bytes = (size_t)rows * kp_;
      uint8_t* x = static_cast<uint8_t*>(scratch_.get(bytes + sizeof(float) * rows));
      float* xs = reinterpret_cast<float*>(x + bytes);
      k::RmsNormArgs a;
      a.x = in.data;
      a.in = in.dtype;
      a.y = x;
      a.out = MNN_E4M3;
      a.scales = xs;
      a.rows = rows;
      a.F = in_;
      a.ldy = kp_;
      k::rmsnorm(ctx(s), a);
      g.x = x;
      g.xs = xs;
    } else if (kp_ != in_ && rows > k::kLinearFew) {  // rows that do not fill the last depth step
      uint8_t* x = static_cast<uint8_t*>(scratch_.get((size_t)rows * kp_));
      k::pad_rows_u8(ctx(s), g.x, rows, in_, x, kp_);
      g.x = x;
    }
    g.w = wq_.as<uint8_t>();
    g.ws = ws_.f32();
    g.bias = b_ ? b_->ptr() : nullptr;
    g.r = res ? res->data : nullptr;
    g.y = out.data;
    g.out = out.dtype;
    g.M = rows;
    g.N = out_;
    g.K = kp_;
    g.ldx = g.x == in.data ? in_ : kp_;
    g.act = act_;
    g.alpha = alpha_;
    k::linear_e4m3(ctx(s), g);
  }

 private:
  void set_weights(const float* data) {
    dev_->make_current();
    DevBuf w;  // the fp32 rows, only while they are rounded
    w.reserve(sizeof(float) * in_ * out_);
    HIP_CHECK(hipMemcpy(w.ptr, data, sizeof(float) * in_ * out_, hipMemcpyHostToDevice));
    k::RmsNormArgs a;
    a.x = w.ptr;
    a.in = MNN_F32;
    a.y = wq_.ptr;
    a.out = MNN_E4M3;
    a.scales = ws_.f32();
    a.rows = out_;
    a.F = in_;
    a.ldy = kp_;
    const LaunchCtx c{dev_, dev_->default_stream};
    k::rmsnorm(c, a);
    HIP_CHECK(hipStreamSynchronize(c.stream));
  }
  int in_, out_, act_, kp_ = 0;
  float alpha_;
  Param* b_ = nullptr;
  DevBuf wq_, ws_;
  Scratch scratch_;
};

// ------------------------------------------------------------------ rotary positions
class RotaryLayer : public ManyInputLayer {
 public:
  RotaryLayer(Device* d, const mnn_rotary_desc& desc) : ManyInputLayer(d), d_(desc) {
    MNN_REQUIRE(desc.head_dim > 0 && desc.head_dim <= 4096, MNN_ERR_INVALID_CONFIGURATION,
                "Rotary: head dim " << desc.head_dim);
    MNN_REQUIRE(desc.num_axes >= 1 && desc.num_axes <= MNN_ROTARY_MAX_AXES,
                MNN_ERR_INVALID_CONFIGURATION, "Rotary: " << desc.num_axes << " axes");
    MNN_REQUIRE(std::isfinite(desc.base) && desc.base > 0.f, MNN_ERR_INVALID_CONFIGURATION,
                "Rotary: base must be finite and positive");
    int64_t sum = 0;
    for (int a = 0; a < desc.num_axes; ++a) {
      const int n = desc.axis_dims[a];
      MNN_REQUIRE(n > 0 && n % 2 == 0, MNN_ERR_INVALID_CONFIGURATION,
                  "Rotary: axis " << a << " turns " << n << " dimensions");
      sum += n;
    }
    MNN_REQUIRE(sum <= desc.head_dim, MNN_ERR_INVALID_CONFIGURATION,
                "Rotary: the axes turn " << sum << " of " << desc.head_dim << " dimensions");
    std::vector<double> rate;
    for (int a = 0; a < desc.num_axes; ++a)
      for (int i = 0; i < desc.axis_dims[a] / 2; ++i)
        rate.push_back(std::pow((double)desc.base, -2.0 * i / desc.axis_dims[a]) /
                       6.283185307179586476925);
    pairs_ = (int)rate.size();
    dev_->make_current();
    rate_.reserve(sizeof(double) * rate.size());
    HIP_CHECK(hipMemcpy(rate_.ptr, rate.data(), sizeof(double) * rate.size(), hipMemcpyHostToDevice));
  }
  const char* kind() const override { return "Rotary"; }
  Shape input_shape() const override { return {0, 0}; }
  Shape output_shape() const override { return {0, 0}; }
  void run(const Tensor& q, const Tensor* kt, const Tensor& pos, Tensor& qo, Tensor* ko, Stream& s) {
    k::RotaryArgs a;
    MNN_REQUIRE((kt != nullptr) == (ko != nullptr), MNN_ERR_INVALID_ARGUMENT,
                "Rotary: k and its output go together");
    MNN_REQUIRE(is_float(q) && (!kt || kt->dtype == q.dtype), MNN_ERR_INVALID_ARGUMENT,
                "Rotary: q and k must both be f32 or both bf16");
    MNN_REQUIRE(pos.dtype == MNN_I32, MNN_ERR_INVALID_ARGUMENT, "Rotary: positions must be i32");
    const Tensor* in[2] = {&q, kt};
    Tensor* out[2] = {&qo, ko};
    for (int i = 0; i < 2 && in[i]; ++i) {
      int64_t B, S, n;
      split_heads("Rotary", in[i]->shape, d_.head_dim, B, S, n);
      MNN_REQUIRE(i == 0 || (B == a.B && S == a.S), MNN_ERR_SHAPE_MISMATCH,
                  "Rotary: k is " << shape_str(kt->shape) << " beside q " << shape_str(q.shape));
      MNN_REQUIRE(n <= 65535, MNN_ERR_INVALID_CONFIGURATION, "Rotary: " << n << " heads");
      MNN_REQUIRE(out[i]->dtype == in[i]->dtype, MNN_ERR_INVALID_ARGUMENT,
                  "Rotary: an output has its input's type");
      MNN_REQUIRE(out[i]->count() == in[i]->count(), MNN_ERR_BUFFER_SIZE_MISMATCH,
                  "Rotary: output " << shape_str(out[i]->shape) << " of "
                                    << shape_str(in[i]->shape));
      a.B = B;
      a.S = S;
      a.heads[i] = (int)n;
      a.x[i] = in[i]->data;
      a.y[i] = out[i]->data;
    }
    MNN_REQUIRE(!same(&qo, kt) && !same(ko, &q) && !same(&qo, ko) && !same(&pos, &qo) &&
                    !same(&pos, ko),
                MNN_ERR_INVALID_ARGUMENT, "Rotary: an output is another argument");
    MNN_REQUIRE(pos.count() == a.S * d_.num_axes || pos.count() == a.B * a.S * d_.num_axes,
                MNN_ERR_BUFFER_SIZE_MISMATCH,
                "Rotary: positions " << shape_str(pos.shape) << " for " << a.B << " x " << a.S
                                     << " tokens and " << d_.num_axes << " axes");
    MNN_REQUIRE(pos.shape.back() == d_.num_axes, MNN_ERR_SHAPE_MISMATCH,
                "Rotary: positions " << shape_str(pos.shape) << " for " << d_.num_axes << " axes");
    a.type = q.dtype;
    a.pos = static_cast<const int*>(pos.data);
    a.shared = pos.count() == a.S * d_.num_axes;
    a.hd = d_.head_dim;
    a.axes = d_.num_axes;
    a.interleaved = d_.interleaved != 0;
    std::copy(d_.axis_dims, d_.axis_dims + d_.num_axes, a.dims);
    a.pairs = pairs_;
    a.rate = rate_.as<double>();
    if (a.B * a.S == 0) return;
    k::rotary(ctx(s), a);
  }

 private:
  mnn_rotary_desc d_;
  int pairs_ = 0;
  DevBuf rate_;
};

// ------------------------------------------------------------------ window attention
class WindowAttentionLayer : public ManyInputLayer {
 public:
  WindowAttentionLayer(Device* d, const mnn_window_attention_desc& desc)
      : ManyInputLayer(d), d_(desc) {
    MNN_REQUIRE(desc.num_heads > 0 && desc.num_kv_heads > 0 && desc.num_heads <= 65535 &&
                    desc.num_heads % desc.num_kv_heads == 0,
                MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: " << desc.num_heads << " heads on " << desc.num_kv_heads);
    MNN_REQUIRE(desc.head_dim > 0 && desc.head_dim % 8 == 0 && desc.head_dim <= 128,
                MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: head dim " << desc.head_dim << " is no multiple of 8 up to 128");
    constexpr int kMost = 1 << 30;
    MNN_REQUIRE(desc.window_left >= 0 && desc.window_left <= kMost && desc.window_right >= 0 &&
                    desc.window_right <= kMost && desc.sinks >= 0 && desc.sinks <= kMost,
                MNN_ERR_INVALID_CONFIGURATION, "WindowAttention: window and sinks must be 0..2^30");
    MNN_REQUIRE(std::isfinite(desc.scale), MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: scale must be finite");
    if (d_.scale == 0.f) d_.scale = 1.f / std::sqrt((float)desc.head_dim);
  }
  const char* kind() const override { return "WindowAttention"; }
  Shape input_shape() const override { return {0, (int64_t)d_.num_heads * d_.head_dim}; }
  Shape output_shape() const override { return input_shape(); }
  void run(const Tensor& q, const Tensor& kt, const Tensor& v, const Tensor* lengths, Tensor& out,
           Stream& s) {
    int64_t B, S;
    check_qkv(q, kt, v, out, B, S);
    MNN_REQUIRE(!lengths || lengths->dtype == MNN_I32, MNN_ERR_INVALID_ARGUMENT,
                "WindowAttention: lengths must be i32");
    MNN_REQUIRE(!lengths || lengths->count() == B, MNN_ERR_BUFFER_SIZE_MISMATCH,
                "WindowAttention: " << lengths->count() << " lengths for a batch of " << B);
    MNN_REQUIRE(!same(lengths, &out), MNN_ERR_INVALID_ARGUMENT,
                "WindowAttention: output is an input");
    if (B * S == 0) return;
    k::WindowArgs a;
    a.q = q.data;
    a.k = kt.data;
    a.v = v.data;
    a.o = out.data;
    a.type = q.dtype;
    a.lengths = lengths ? static_cast<const int*>(lengths->data) : nullptr;
    a.B = (int)B;
    a.S = (int)S;
    a.H = d_.num_heads;
    a.KV = d_.num_kv_heads;
    a.hd = d_.head_dim;
    a.left = d_.window_left;
    a.right = d_.window_right;
    a.sinks = d_.sinks;
    a.scale = d_.scale;
    k::window_attention(ctx(s), a);
  }
  void step(const Tensor& q, const Tensor& kt, const Tensor& v, const Tensor& pos, const Tensor* steps,
            Tensor& kc, Tensor& vc, Tensor& out, Stream& s) {
    MNN_REQUIRE(d_.window_right == 0, MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: a step has no tokens to come (window_right "
                    << d_.window_right << ")");
    int64_t B, T;
    check_qkv(q, kt, v, out, B, T);
    MNN_REQUIRE(T <= 65535, MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: " << T << " new tokens in one step, at most 65535");
    const int64_t kvw = (int64_t)d_.num_kv_heads * d_.head_dim;
    for (const Tensor* c : {&kc, &vc}) {
      MNN_REQUIRE(c->dtype == q.dtype, MNN_ERR_INVALID_ARGUMENT,
                  "WindowAttention: the caches have the type of q");
      MNN_REQUIRE(c->shape.size() == 3 && c->shape[0] == B && c->shape[2] == kvw &&
                      c->shape == kc.shape,
                  MNN_ERR_SHAPE_MISMATCH, "WindowAttention: cache " << shape_str(c->shape)
                                              << ", expected [" << B << ", slots, " << kvw << "]");
    }
    const int64_t C = kc.shape[1], need = (int64_t)d_.sinks + d_.window_left + T;
    MNN_REQUIRE(C >= need && C <= (1 << 30), MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: " << C << " cache slots, " << need << " needed (sinks + window_left + "
                                    << T << " new tokens), at most 2^30");
    for (const Tensor* t : {&pos, steps})
      if (t) {
        MNN_REQUIRE(t->dtype == MNN_I32, MNN_ERR_INVALID_ARGUMENT,
                    "WindowAttention: positions and steps must be i32");
        MNN_REQUIRE(t->count() == B, MNN_ERR_BUFFER_SIZE_MISMATCH,
                    "WindowAttention: " << t->count() << " positions or steps for a batch of " << B);
      }
    const Tensor* written[3] = {&kc, &vc, &out};
    for (int i = 0; i < 3; ++i) {
      for (const Tensor* t : {&q, &kt, &v, &pos, steps})
        MNN_REQUIRE(!same(written[i], t), MNN_ERR_INVALID_ARGUMENT,
                    "WindowAttention: an output or cache is an input");
      for (int j = 0; j < i; ++j)
        MNN_REQUIRE(!same(written[i], written[j]), MNN_ERR_INVALID_ARGUMENT,
                    "WindowAttention: output and caches must be three tensors");
    }
    if (B * T == 0) return;
    k::WindowStepArgs a;
    a.q = q.data;
    a.k = kt.data;
    a.v = v.data;
    a.kc = kc.data;
    a.vc = vc.data;
    a.o = out.data;
    a.type = q.dtype;
    a.pos = static_cast<const int*>(pos.data);
    a.steps = steps ? static_cast<const int*>(steps->data) : nullptr;
    a.B = (int)B;
    a.T = (int)T;
    a.C = (int)C;
    a.H = d_.num_heads;
    a.KV = d_.num_kv_heads;
    a.hd = d_.head_dim;
    a.left = d_.window_left;
    a.sinks = d_.sinks;
    a.scale = d_.scale;
    const int64_t part = k::window_step_part_floats(ctx(s), a);
    k::window_step(ctx(s), a, part ? static_cast<float*>(scratch_.get(sizeof(float) * part)) : nullptr);
  }

 private:
  void check_qkv(const Tensor& q, const Tensor& kt, const Tensor& v, const Tensor& out, int64_t& B,
                 int64_t& S) const {
    int64_t n, b, t;
    split_heads("WindowAttention", q.shape, d_.head_dim, B, S, n);
    MNN_REQUIRE(n == d_.num_heads, MNN_ERR_SHAPE_MISMATCH,
                "WindowAttention: q " << shape_str(q.shape) << " has " << n << " heads, expected "
                                      << d_.num_heads);
    for (const Tensor* x : {&kt, &v}) {
      split_heads("WindowAttention", x->shape, d_.head_dim, b, t, n);
      MNN_REQUIRE(b == B && t == S && n == d_.num_kv_heads, MNN_ERR_SHAPE_MISMATCH,
                  "WindowAttention: k or v " << shape_str(x->shape) << " beside q "
                                             << shape_str(q.shape));
    }
    MNN_REQUIRE(is_float(q) && kt.dtype == q.dtype && v.dtype == q.dtype && out.dtype == q.dtype,
                MNN_ERR_INVALID_ARGUMENT,
                "WindowAttention: q, k, v and output must all be f32 or all bf16");
    MNN_REQUIRE(out.count() == q.count(), MNN_ERR_BUFFER_SIZE_MISMATCH,
                "WindowAttention: output " << shape_str(out.shape) << " for q "
                                           << shape_str(q.shape));
    MNN_REQUIRE(B <= 65535 && S <= (1 << 30), MNN_ERR_INVALID_CONFIGURATION,
                "WindowAttention: batch " << B << " or length " << S << " too large");
    MNN_REQUIRE(!same(&out, &q) && !same(&out, &kt) && !same(&out, &v), MNN_ERR_INVALID_ARGUMENT,
                "WindowAttention: output is an input");
  }
  mnn_window_attention_desc d_;
  Scratch scratch_;
};

}  // namespace

std::unique_ptr<Layer> make_rmsnorm(Device* d, int features, float eps) {
  return std::make_unique<RMSNormLayer>(d, features, eps);
}
void rmsnorm_forward_residual(Layer* l, const Tensor& in, const Tensor* res, Tensor* sum, Tensor& out,
                              Tensor* scales, Stream& s) {
  as<RMSNormLayer>(l, "mnn_rmsnorm_forward_residual").run(in, res, sum, out, scales, s);
}

std::unique_ptr<Layer> make_linear_e4m3(Device* d, int in, int out, bool bias, int act,
                                        float leaky_alpha) {
  return std::make_unique<LinearE4m3Layer>(d, in, out, bias, act, leaky_alpha);
}
void linear_forward_scaled(Layer* l, const Tensor& in, const Tensor* scales, const Tensor* res,
                           Tensor& out, Stream& s) {
  as<LinearE4m3Layer>(l, "mnn_linear_forward_scaled (precision e4m3)").run(in, scales, res, out, s);
}

std::unique_ptr<Layer> make_rotary(Device* d, const mnn_rotary_desc& desc) {
  return std::make_unique<RotaryLayer>(d, desc);
}
void rotary_forward(Layer* l, const Tensor& q, const Tensor* kt, const Tensor& pos, Tensor& q_out,
                    Tensor* k_out, Stream& s) {
  as<RotaryLayer>(l, "mnn_rotary_forward").run(q, kt, pos, q_out, k_out, s);
}

std::unique_ptr<Layer> make_window_attention(Device* d, const mnn_window_attention_desc& desc) {
  return std::make_unique<WindowAttentionLayer>(d, desc);
}
void window_attention_forward(Layer* l, const Tensor& q, const Tensor& kt, const Tensor& v,
                              const Tensor* lengths, Tensor& out, Stream& s) {
  as<WindowAttentionLayer>(l, "mnn_window_attention_forward").run(q, kt, v, lengths, out, s);
}
void window_attention_step(Layer* l, const Tensor& q, const Tensor& kt, const Tensor& v,
                           const Tensor& pos, const Tensor* steps, Tensor& k_cache, Tensor& v_cache,
                           Tensor& out, Stream& s) {
  as<WindowAttentionLayer>(l, "mnn_window_attention_step")
      .step(q, kt, v, pos, steps, k_cache, v_cache, out, s);
}

}  // namespace mnn
