// extern "C" boundary of the operators around dispatch and combine (rows to 8 bits and back, the experts'
// products, the layer for a few tokens): argument checks on the host, then kernel launches.  No allocation,
// no synchronisation and no state; none of these calls depends on shapes fixed at build time.
#include "../../include/mi_ep.h"

#include "ep_expert.h"

namespace {

using namespace mi_ep;

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }
inline int status_of(hipError_t e) { return e == hipSuccess ? MI_EP_OK : static_cast<int>(e); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// Rows of the 8-bit formats; the scales' strides count floats.
inline bool quantized_shape_ok(int num_rows, int hidden, int format, long long scales_row_stride,
                               long long scales_hidden_stride) {
  if (num_rows < 0 || num_rows >= (1 << 30) || hidden <= 0 || hidden % 8 != 0 || hidden > MI_EP_QUANT_MAX_HIDDEN) return false;
  if (format != MI_EP_QUANT_INT8_ROW && format != MI_EP_QUANT_E4M3_BLOCK) return false;
  if (format == MI_EP_QUANT_E4M3_BLOCK && hidden % MI_EP_QUANT_BLOCK != 0) return false;
  return scales_row_stride >= 0 && (format == MI_EP_QUANT_INT8_ROW || scales_hidden_stride >= 0);
}
// Written scales: every one has a place of its own.
inline bool scales_distinct(int num_rows, int hidden, int format, long long row_stride, long long hidden_stride) {
  const long long groups = format == MI_EP_QUANT_INT8_ROW ? 1 : hidden / MI_EP_QUANT_BLOCK;
  if (num_rows > 1 && row_stride < 1) return false;
  if (groups > 1 && hidden_stride < 1) return false;
  if (num_rows <= 1 || groups <= 1) return true;
  return row_stride >= (groups - 1) * hidden_stride + 1 || hidden_stride >= (num_rows - 1) * row_stride + 1;
}
inline bool row_stride_ok(long long stride, int hidden) { return stride >= hidden && stride % 8 == 0; }
// Whether written rows, one behind the other, lie across others' rows of the same width: a workgroup would write what
// another one has yet to read.  The same rows (in place) do not.
inline bool written_across(const void* written, const void* read, long long read_stride, int num_rows, int hidden) {
  const long long out = reinterpret_cast<long long>(written), in = reinterpret_cast<long long>(read);
  const long long width = 2LL * hidden, stride = 2 * read_stride;
  if (num_rows == 0 || (out == in && stride == width)) return false;
  const long long first = in + width > out ? 0 : (out - in - width) / stride + 1;  // the first row that ends behind `out`
  return first < num_rows && in + first * stride < out + num_rows * width;
}

inline bool few_tokens_shape_ok(int num_tokens, int num_topk) {
  return num_tokens >= 0 && num_topk > 0 && num_topk <= MI_EP_MAX_TOPK &&
         static_cast<long long>(num_tokens) * num_topk <= MI_EP_FEW_MAX_ROUTES;
}

}  // namespace

extern "C" {

int mi_ep_rms_norm_quantize(const void* x, long long x_row_stride, const void* residual,
                            long long residual_row_stride, const void* weight, unsigned int epsilon_bits,
                            int num_rows, int hidden, int format, void* q, float* scales,
                            long long scales_row_stride, long long scales_hidden_stride, void* residual_out,
                            void* normed, void* stream) {
  const float eps = __builtin_bit_cast(float, epsilon_bits);
  if (!(eps >= 0.0f && eps < __builtin_inff())) return MI_EP_EINVAL;
  if (!quantized_shape_ok(num_rows, hidden, format, scales_row_stride, scales_hidden_stride)) return MI_EP_EINVAL;
  if (!scales_distinct(num_rows, hidden, format, scales_row_stride, scales_hidden_stride)) return MI_EP_EINVAL;
  if (!row_stride_ok(x_row_stride, hidden) || (residual != nullptr && !row_stride_ok(residual_row_stride, hidden)))
    return MI_EP_EINVAL;
  if (residual_out != nullptr && residual == nullptr) return MI_EP_EINVAL;
  if (residual_out != nullptr && (written_across(residual_out, x, x_row_stride, num_rows, hidden) ||
                                  written_across(residual_out, residual, residual_row_stride, num_rows, hidden)))
    return MI_EP_EINVAL;
  if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(residual_out) || !aligned16(normed) ||
      !aligned8(q))
    return MI_EP_EINVAL;
  if (num_rows > 0 && (x == nullptr || weight == nullptr || q == nullptr || scales == nullptr)) return MI_EP_EINVAL;

  QuantizeArgs a{};
  a.x = static_cast<const vec16*>(x);
  a.residual = static_cast<const vec16*>(residual);
  a.weight = static_cast<const vec16*>(weight);
  a.q = static_cast<uint2*>(q);
  a.scales = scales;
  a.residual_out = static_cast<vec16*>(residual_out);
  a.normed = static_cast<vec16*>(normed);
  a.x_row_vecs = x_row_stride / 8;
  a.residual_row_vecs = residual_row_stride / 8;
  a.scales_row_stride = scales_row_stride;
  a.scales_hidden_stride = scales_hidden_stride;
  a.num_rows = num_rows;
  a.row_vecs = hidden / 8;
  a.eps = eps;
  return status_of(launch_quantize_rows(a, format, as_stream(stream)));
}

int mi_ep_quantize_rows(const void* x, long long x_row_stride, const int* row_limit, int num_rows, int hidden,
                        int format, void* q, float* scales, long long scales_row_stride,
                        long long scales_hidden_stride, void* stream) {
  if (!quantized_shape_ok(num_rows, hidden, format, scales_row_stride, scales_hidden_stride)) return MI_EP_EINVAL;
  if (!scales_distinct(num_rows, hidden, format, scales_row_stride, scales_hidden_stride)) return MI_EP_EINVAL;
  if (!row_stride_ok(x_row_stride, hidden) || !aligned16(x) || !aligned8(q)) return MI_EP_EINVAL;
  if (num_rows > 0 && (x == nullptr || q == nullptr || scales == nullptr)) return MI_EP_EINVAL;
  QuantizeArgs a{};
  a.x = static_cast<const vec16*>(x);
  a.row_limit = row_limit;
  a.q = static_cast<uint2*>(q);
  a.scales = scales;
  a.x_row_vecs = x_row_stride / 8;
  a.scales_row_stride = scales_row_stride;
  a.scales_hidden_stride = scales_hidden_stride;
  a.num_rows = num_rows;
  a.row_vecs = hidden / 8;
  return status_of(launch_quantize_rows(a, format, as_stream(stream)));
}

int mi_ep_dequantize_rows(const void* q, const float* scales, long long scales_row_stride,
                          long long scales_hidden_stride, const int* row_limit, int num_rows, int hidden,
                          int format, void* out, void* stream) {
  if (!quantized_shape_ok(num_rows, hidden, format, scales_row_stride, scales_hidden_stride)) return MI_EP_EINVAL;
  if (!aligned8(q) || !aligned16(out)) return MI_EP_EINVAL;
  if (num_rows > 0 && (q == nullptr || scales == nullptr || out == nullptr)) return MI_EP_EINVAL;
  DequantizeArgs a{};
  a.q = static_cast<const uint2*>(q);
  a.scales = scales;
  a.row_limit = row_limit;
  a.out = static_cast<vec16*>(out);
  a.scales_row_stride = scales_row_stride;
  a.scales_hidden_stride = scales_hidden_stride;
  a.num_rows = num_rows;
  a.row_vecs = hidden / 8;
  return status_of(launch_dequantize_rows(a, format, as_stream(stream)));
}

int mi_ep_grouped_matmul_int8(const void* a, const float* a_scales, long long a_scales_row_stride, const void* b,
                              const float* b_scales, const int* expert_offsets,
                              const int* num_tokens_per_expert, int num_rows, int num_experts, int out_features,
                              int in_features, void* out, int flags, void* stream) {
  const bool silu_mul = (flags & MI_EP_MATMUL_SILU_MUL) != 0;
  if ((flags & ~MI_EP_MATMUL_SILU_MUL) != 0) return MI_EP_EINVAL;
  if (num_rows < 0 || num_rows >= (1 << 28) || num_experts <= 0 || num_experts > MI_EP_MAX_EXPERTS) return MI_EP_EINVAL;
  // |a * b| <= 2^14: 2^17 of them are the most whose sum is sure to fit 32 bits.
  if (in_features <= 0 || in_features % 16 != 0 || in_features >= (1 << 17)) return MI_EP_EINVAL;
  if (out_features <= 0 || out_features % (silu_mul ? 16 : 8) != 0 || out_features > (1 << 20)) return MI_EP_EINVAL;
  // Tiles of the product are counted in int.
  if ((num_rows / 256 + num_experts) * (out_features / 128 + 1LL) >= (1LL << 31)) return MI_EP_EINVAL;
  if (a_scales_row_stride < 0 || a_scales_row_stride > (1 << 20)) return MI_EP_EINVAL;  // a tile's scales lie within 2^30 bytes
  if (expert_offsets == nullptr && (num_experts != 1 || num_tokens_per_expert != nullptr)) return MI_EP_EINVAL;
  if (!aligned16(a) || !aligned16(b) || !aligned16(out)) return MI_EP_EINVAL;
  if (num_rows > 0 && (a == nullptr || a_scales == nullptr || b == nullptr || b_scales == nullptr || out == nullptr))
    return MI_EP_EINVAL;
  ExpertMatmulArgs m{};
  m.a = static_cast<const unsigned char*>(a);
  m.a_scales = a_scales;
  m.b = static_cast<const unsigned char*>(b);
  m.b_scales = b_scales;
  m.expert_offsets = expert_offsets;
  m.num_tokens_per_expert = num_tokens_per_expert;
  m.out = static_cast<uint16_t*>(out);
  m.a_scales_row_stride = a_scales_row_stride;
  m.num_rows = num_rows;
  m.num_experts = num_experts;
  m.out_features = out_features;
  m.in_features = in_features;
  m.silu_mul = silu_mul ? 1 : 0;
  return status_of(launch_expert_matmul(m, as_stream(stream)));
}

size_t mi_ep_moe_few_tokens_workspace_bytes(int num_tokens, int num_topk, int hidden, int intermediate) {
  if (!few_tokens_shape_ok(num_tokens, num_topk) || intermediate <= 0 || intermediate % 16 != 0 || intermediate > 65536 ||
      hidden <= 0 || hidden % 16 != 0 || hidden > 65536)
    return 0;
  return static_cast<size_t>(num_tokens) * num_topk * (static_cast<size_t>(intermediate) + hidden) * 4;
}

int mi_ep_moe_few_tokens(const void* x, const int64_t* topk_idx, const float* topk_weights, const void* w13,
                         const float* w13_scales, const void* w2, const float* w2_scales, const void* bias_0,
                         const void* bias_1, int num_tokens, int num_topk, int num_experts, int hidden,
                         int intermediate, void* combined_x, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (!few_tokens_shape_ok(num_tokens, num_topk) || num_experts <= 0 || num_experts > MI_EP_MAX_EXPERTS) return MI_EP_EINVAL;
  if (hidden <= 0 || hidden % 16 != 0 || hidden > 65536) return MI_EP_EINVAL;
  if (intermediate <= 0 || intermediate % 16 != 0 || intermediate > 65536) return MI_EP_EINVAL;
  if ((w13_scales != nullptr) != (w2_scales != nullptr)) return MI_EP_EINVAL;
  if (!aligned16(x) || !aligned16(w13) || !aligned16(w2) || !aligned16(bias_0) || !aligned16(bias_1) ||
      !aligned16(combined_x) || !aligned16(workspace))
    return MI_EP_EINVAL;
  if (num_tokens == 0) return MI_EP_OK;
  if (x == nullptr || topk_idx == nullptr || w13 == nullptr || w2 == nullptr || combined_x == nullptr || workspace == nullptr)
    return MI_EP_EINVAL;
  if (workspace_bytes < mi_ep_moe_few_tokens_workspace_bytes(num_tokens, num_topk, hidden, intermediate)) return MI_EP_ENOSPC;
  FewTokensArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.topk_idx = topk_idx;
  a.topk_weights = topk_weights;
  a.w13 = static_cast<const unsigned char*>(w13);
  a.w2 = static_cast<const unsigned char*>(w2);
  a.w13_scales = w13_scales;
  a.w2_scales = w2_scales;
  a.bias_0 = static_cast<const uint16_t*>(bias_0);
  a.bias_1 = static_cast<const uint16_t*>(bias_1);
  a.act = static_cast<uint16_t*>(workspace);
  a.y = reinterpret_cast<float*>(a.act + static_cast<size_t>(num_tokens) * num_topk * intermediate * 2);
  a.combined_x = static_cast<uint16_t*>(combined_x);
  a.num_tokens = num_tokens;
  a.num_topk = num_topk;
  a.num_experts = num_experts;
  a.hidden = hidden;
  a.intermediate = intermediate;
  return status_of(launch_few_tokens(a, as_stream(stream)));
}

}  // extern "C"
