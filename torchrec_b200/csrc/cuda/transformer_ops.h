// Host functions of the transformer kernels that the autograd layer calls (transformer_autograd.cpp).
#pragma once

#include <ATen/ATen.h>

#include <tuple>

namespace trb {

// full_softmax_kernels.cu
std::tuple<at::Tensor, at::Tensor> full_softmax_fwd(const at::Tensor& h, const at::Tensor& weight, const at::Tensor& targets, const c10::optional<at::Tensor>& bias,
                                                    int64_t ignore_index, int64_t reduction, int64_t grad, int64_t gave_up);
std::tuple<at::Tensor, at::Tensor, at::Tensor> full_softmax_bwd(const at::Tensor& dloss, const at::Tensor& weight, const at::Tensor& state, int64_t P, int64_t D, bool has_bias,
                                                                int64_t reduction, bool has_unit, bool want_h, bool want_w, bool want_b, bool dh_fp32, bool dw_fp32, bool db_fp32);

// rotary_kernels.cu
at::Tensor qk_norm_rotary_fwd(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq, const c10::optional<at::Tensor>& qw,
                              const c10::optional<at::Tensor>& kw, at::IntArrayRef sections, int64_t heads, int64_t kv_heads, double eps, bool norm, bool interleaved);
std::tuple<at::Tensor, at::Tensor> qk_norm_rotary_bwd(const at::Tensor& dy, const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq,
                                                      const c10::optional<at::Tensor>& qw, const c10::optional<at::Tensor>& kw, at::IntArrayRef sections, int64_t heads,
                                                      int64_t kv_heads, double eps, bool norm, bool interleaved, bool want_dw);

}  // namespace trb
