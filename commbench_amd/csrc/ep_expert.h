// Launcher declarations and device helpers of the operators around dispatch and combine: rows to 8 bits and back, the
// experts' products, the layer for a few tokens.
#pragma once

#include "ep_device.h"

namespace mi_ep {

// ---- rows to 8 bits and back ----------------------------------------------------
constexpr int kQuantInt8 = 0;    // one scale per row
constexpr int kQuantE4m3 = 1;    // one scale per kQuantBlock columns
constexpr int kQuantBlock = 128;
constexpr int kQuantMaxVecs = 4096;  // a row stays in one workgroup's registers: up to 32768 columns

struct QuantizeArgs {
  const vec16* x;         // bf16 rows, 8 columns per vector
  const vec16* residual;  // bf16 rows added first, or null
  const vec16* weight;    // bf16 [hidden]: the norm's gain; null = no norm
  const int* row_limit;   // null, or a device word: rows at and beyond it are left as they are
  uint2* q;               // 8 codes per word pair
  float* scales;
  vec16* residual_out;    // x + residual, or null
  vec16* normed;          // the rows before quantisation, or null
  long long x_row_vecs, residual_row_vecs;  // vectors between rows
  long long scales_row_stride, scales_hidden_stride;  // in floats
  int num_rows;
  int row_vecs;
  int first_row;  // of the launch; set by the launcher
  float eps;
};
hipError_t launch_quantize_rows(const QuantizeArgs& a, int format, hipStream_t stream);

struct DequantizeArgs {
  const uint2* q;
  const float* scales;
  const int* row_limit;
  vec16* out;
  long long scales_row_stride, scales_hidden_stride;
  int num_rows;
  int row_vecs;
  bool stream_output;  // set by the launcher
};
hipError_t launch_dequantize_rows(const DequantizeArgs& a, int format, hipStream_t stream);

// ---- the experts' products --------------------------------------------------------
struct ExpertMatmulArgs {
  const unsigned char* a;  // int8 [num_rows, in_features]
  const float* a_scales;   // per row, a_scales_row_stride floats apart
  const unsigned char* b;  // int8 [num_experts, out_features, in_features]
  const float* b_scales;   // [num_experts, out_features]
  const int* expert_offsets;         // [num_experts + 1], or null: one expert owns all rows
  const int* num_tokens_per_expert;  // [num_experts] or null: whole segments are rows
  uint16_t* out;                     // bf16 [num_rows, out_features, or half of it with silu_mul]
  long long a_scales_row_stride;
  int num_rows;
  int num_experts;
  int out_features;
  int in_features;
  int silu_mul;
};
hipError_t launch_expert_matmul(const ExpertMatmulArgs& a, hipStream_t stream);

constexpr int kFewRoutes = 1024;  // routes of one launch: their products are collected in LDS
struct FewTokensArgs {
  const uint16_t* x;  // bf16 [num_tokens, hidden]
  const int64_t* topk_idx;
  const float* topk_weights;  // or null: a plain sum
  const unsigned char* w13;   // [num_experts, 2 * intermediate, hidden]: gate rows, then up rows
  const unsigned char* w2;    // [num_experts, hidden, intermediate]
  const float* w13_scales;    // [num_experts, 2 * intermediate] with int8 weights, null with bf16
  const float* w2_scales;     // [num_experts, hidden]
  const uint16_t* bias_0;
  const uint16_t* bias_1;
  uint16_t* act;  // bf16 [2, num_tokens * num_topk, intermediate]: two terms of every value
  float* y;       // [num_tokens * num_topk, hidden]: the products of every route, where a sum of its own adds them
  uint16_t* combined_x;
  int num_tokens;
  int num_topk;
  int num_experts;
  int hidden;
  int intermediate;
};
hipError_t launch_few_tokens(const FewTokensArgs& a, hipStream_t stream);

#ifdef __HIPCC__
// Two values to bf16, nearest even, in the conversion instruction.
__device__ __forceinline__ uint32_t to_bf16_pair(float lo, float hi) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  union {
    bf16x2 b;
    uint32_t u;
  } out;
  out.b = __builtin_convertvector((float2v{lo, hi}), bf16x2);
  return out.u;
}
#endif

}  // namespace mi_ep
