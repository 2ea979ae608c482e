// Layers over tokens beside those of the MetalNN stack: RMSNorm with residual and 8-bit output, the
// 8-bit Linear that reads it, rotary positions, window attention, rolling caches, attention to an
// encoder's states. Entry points that take more than one
// input are free functions on a Layer*, refused for layers of another kind.
#pragma once

#include "layers.hpp"

namespace mnn {

std::unique_ptr<Layer> make_rmsnorm(Device* d, int features, float eps);
void rmsnorm_forward_residual(Layer* l, const Tensor& in, const Tensor* res, Tensor* sum, Tensor& out,
                              Tensor* scales, Stream& s);

std::unique_ptr<Layer> make_linear_e4m3(Device* d, int in, int out, bool bias, int act,
                                        float leaky_alpha, bool blocks);
void linear_forward_scaled(Layer* l, const Tensor& in, const Tensor* scales, const Tensor* res,
                           Tensor& out, Stream& s);

std::unique_ptr<Layer> make_rotary(Device* d, const mnn_rotary_desc& desc);
void rotary_forward(Layer* l, const Tensor& q, const Tensor* k, const Tensor& pos, Tensor& q_out,
                    Tensor* k_out, Stream& s);

std::unique_ptr<Layer> make_window_attention(Device* d, const mnn_window_attention_desc& desc);
void window_attention_forward(Layer* l, const Tensor& q, const Tensor& k, const Tensor& v,
                              const Tensor* lengths, Tensor& out, Stream& s);
void window_attention_step(Layer* l, const Tensor& q, const Tensor& k, const Tensor& v,
                           const Tensor& pos, const Tensor* steps, Tensor& k_cache, Tensor& v_cache,
                           Tensor& out, Stream& s);
void window_attention_step_e4m3(Layer* l, const Tensor& q, const Tensor& k, const Tensor& v,
                                const Tensor& pos, const Tensor* steps, Tensor& k_cache,
                                Tensor& k_scales, Tensor& v_cache, Tensor& v_scales, Tensor& out,
                                Stream& s);

std::unique_ptr<Layer> make_kv_cache(Device* d, int kv_heads, int head_dim, int sinks);
void kv_cache_write(Layer* l, const Tensor& k, const Tensor& v, const Tensor& pos, const Tensor* steps,
                    Tensor& k_cache, Tensor* k_scales, Tensor& v_cache, Tensor* v_scales, Stream& s);
void kv_cache_read(Layer* l, const Tensor& k_cache, const Tensor* k_scales, const Tensor& v_cache,
                   const Tensor* v_scales, const Tensor& pos, const Tensor* steps, Tensor& k, Tensor& v,
                   Stream& s);

std::unique_ptr<Layer> make_memory_attention(Device* d, const mnn_memory_attention_desc& desc);
void memory_attention_forward(Layer* l, const Tensor& q, const Tensor& k, const Tensor* k_scales,
                              const Tensor& v, const Tensor* v_scales, const Tensor* query_lengths,
                              const Tensor* lengths, Tensor& out, Stream& s);

}  // namespace mnn
